"""What batch_inputs, tree_attention and adjust_logits refuse, on tensors that never reach a GPU: every refusal is an error
before anything is launched, and a call that fits gets as far as the check for the GPU."""
import pytest
import torch

I32, I64, F32, BF16 = torch.int32, torch.int64, torch.float32, torch.bfloat16


@pytest.fixture
def ops(pkg, monkeypatch):
    from nanovllm_b200 import ops

    class Runtime:
        handle = None

    monkeypatch.setattr(ops, "get_runtime", lambda: Runtime)
    return ops


def batch_args(**kw):
    a = dict(block_tables=torch.zeros(3, 4, dtype=I32), cached_lens=torch.zeros(3, dtype=I32), seq_lens=torch.zeros(3, dtype=I32), free_blocks=torch.zeros(9, dtype=I32),
             num_free=torch.zeros(1, dtype=I32), block_size=16, num_slots=160, max_tokens=8, tree_mask=None)
    a.update(kw)
    return a


STACK = torch.zeros(12, dtype=I32)


@pytest.mark.parametrize("error, change", [
    (ValueError, dict(block_tables=torch.zeros(12, dtype=I32))),
    (TypeError, dict(block_tables=torch.zeros(3, 4, dtype=I64))),
    (AssertionError, dict(block_tables=torch.zeros(4, 3, dtype=I32).t())),
    (AssertionError, dict(block_tables=torch.zeros(1, 4, dtype=I32).expand(3, 4))),
    (ValueError, dict(block_tables=torch.zeros(3, 0, dtype=I32))),
    (ValueError, dict(cached_lens=torch.zeros(2, dtype=I32))),
    (TypeError, dict(cached_lens=torch.zeros(3, dtype=I64))),
    (AssertionError, dict(seq_lens=torch.zeros(6, dtype=I32)[::2])),
    (ValueError, dict(seq_lens=torch.zeros(3, 1, dtype=I32))),
    (TypeError, dict(free_blocks=torch.zeros(9, dtype=F32))),
    (ValueError, dict(num_free=torch.zeros(2, dtype=I32))),
    (ValueError, dict(block_size=0)),
    (ValueError, dict(num_slots=0)),
    (ValueError, dict(max_tokens=-1)),
    (ValueError, dict(block_size=1 << 29)),
    (ValueError, dict(tree_mask=torch.zeros(7, 1, dtype=I64))),
    (ValueError, dict(tree_mask=torch.zeros(8, 0, dtype=I64))),
    (TypeError, dict(tree_mask=torch.zeros(8, 1, dtype=I32))),
    (AssertionError, dict(tree_mask=torch.zeros(1, 2, dtype=I64).expand(8, 2))),
    (ValueError, dict(block_tables=STACK.view(3, 4), free_blocks=STACK)),
    (ValueError, dict(free_blocks=STACK, num_free=STACK[:1])),
    (ValueError, dict(block_tables=torch.zeros(8193, 1, dtype=I32), cached_lens=torch.zeros(8193, dtype=I32), seq_lens=torch.zeros(8193, dtype=I32))),
])
def test_batch_inputs_refusals(ops, error, change):
    with pytest.raises(error):
        ops.batch_inputs(**batch_args(**change))


@pytest.mark.parametrize("change", [{}, dict(tree_mask=torch.zeros(9, 2, dtype=I64)), dict(block_tables=torch.zeros(3, 6, dtype=I32)[:, 1:5]), dict(free_blocks=torch.zeros(0, dtype=I32)),
                                    dict(block_tables=torch.zeros(0, 4, dtype=I32), cached_lens=torch.zeros(0, dtype=I32), seq_lens=torch.zeros(0, dtype=I32))])
def test_batch_inputs_that_fit_need_a_gpu(ops, change):
    with pytest.raises(TypeError, match="GPU"):
        ops.batch_inputs(**batch_args(**change))


def tree_args(**kw):
    a = dict(q=torch.zeros(5, 4, 128, dtype=BF16), k_cache=torch.zeros(3, 16, 2, 128, dtype=BF16), v_cache=torch.zeros(3, 16, 2, 128, dtype=BF16),
             cu_seqlens_q=torch.zeros(3, dtype=I32), context_lens=torch.zeros(2, dtype=I32), block_tables=torch.zeros(2, 2, dtype=I32),
             tree_mask=torch.zeros(5, 1, dtype=I64), max_seqlen_q=3, scale=0.1)
    a.update(kw)
    return a


@pytest.mark.parametrize("error, change", [
    (ValueError, dict(q=torch.zeros(5, 512, dtype=BF16))),
    (TypeError, dict(q=torch.zeros(5, 4, 128))),
    (ValueError, dict(q=torch.zeros(5, 3, 128, dtype=BF16))),
    (ValueError, dict(q=torch.zeros(5, 4, 64, dtype=BF16))),
    (ValueError, dict(q=torch.zeros(5, 4, 96, dtype=BF16), k_cache=torch.zeros(3, 16, 2, 96, dtype=BF16), v_cache=torch.zeros(3, 16, 2, 96, dtype=BF16))),
    (ValueError, dict(q=torch.zeros(5, 258, 128, dtype=BF16))),
    (AssertionError, dict(q=torch.zeros(4, 5, 128, dtype=BF16).transpose(0, 1))),
    (AssertionError, dict(q=torch.zeros(5 * 516, dtype=BF16).as_strided((5, 4, 128), (516, 128, 1)))),
    (TypeError, dict(k_cache=torch.zeros(3, 16, 2, 128), v_cache=torch.zeros(3, 16, 2, 128))),
    (ValueError, dict(v_cache=torch.zeros(3, 16, 1, 128, dtype=BF16))),
    (ValueError, dict(k_cache=torch.zeros(3, 24, 2, 128, dtype=BF16), v_cache=torch.zeros(3, 24, 2, 128, dtype=BF16))),
    (AssertionError, dict(k_cache=torch.zeros(3, 2, 16, 128, dtype=BF16).transpose(1, 2))),
    (ValueError, dict(k_cache=torch.zeros(0, 16, 2, 128, dtype=BF16), v_cache=torch.zeros(0, 16, 2, 128, dtype=BF16))),
    (ValueError, dict(cu_seqlens_q=torch.zeros(2, dtype=I32))),
    (TypeError, dict(cu_seqlens_q=torch.zeros(3, dtype=I64))),
    (TypeError, dict(context_lens=torch.zeros(2, dtype=I64))),
    (ValueError, dict(block_tables=torch.zeros(3, 2, dtype=I32))),
    (ValueError, dict(block_tables=torch.zeros(2, 0, dtype=I32))),
    (AssertionError, dict(block_tables=torch.zeros(2, 2, dtype=I32).t())),
    (ValueError, dict(tree_mask=torch.zeros(4, 1, dtype=I64))),
    (ValueError, dict(tree_mask=torch.zeros(5, 0, dtype=I64))),
    (TypeError, dict(tree_mask=torch.zeros(5, 1, dtype=torch.bool))),
    (ValueError, dict(max_seqlen_q=0)),
    (AssertionError, dict(block_tables=torch.zeros(1, 2, dtype=I32).expand(2, 2))),
    (AssertionError, dict(tree_mask=torch.zeros(1, 2, dtype=I64).expand(5, 2))),
    (ValueError, dict(q=torch.zeros(5, 4, 128, dtype=BF16, requires_grad=True))),
])
def test_tree_attention_refusals(ops, error, change):
    with pytest.raises(error):
        ops.tree_attention(**tree_args(**change))


@pytest.mark.parametrize("change", [{}, dict(tree_mask=torch.zeros(5, 3, dtype=I64)), dict(q=torch.zeros(5, 8, 128, dtype=BF16)[:, :4])])
def test_tree_attention_that_fits_needs_a_gpu(ops, change):
    with pytest.raises(TypeError, match="GPU"):
        ops.tree_attention(**tree_args(**change))


def rules(**kw):
    a = dict(logits=torch.zeros(4, 70), history=torch.zeros(2, 9, dtype=I64), history_lens=torch.zeros(2, dtype=I32), prompt_lens=torch.zeros(2, dtype=I32),
             repetition_penalty=torch.ones(2), presence_penalty=torch.ones(2), frequency_penalty=torch.ones(2), bias_ids=torch.zeros(2, 3, dtype=I64),
             bias_values=torch.zeros(2, 3), allowed_mask=torch.zeros(4, 3, dtype=I32), cu_seqlens=torch.zeros(3, dtype=I32),
             draft_tokens=torch.zeros(4, dtype=I64), tree_mask=torch.zeros(4, 1, dtype=I64), out=None)
    a.update(kw)
    return a


ROWS = torch.zeros(5, 70)


@pytest.mark.parametrize("error, change", [
    (ValueError, dict(logits=torch.zeros(280))),
    (TypeError, dict(logits=torch.zeros(4, 70, dtype=torch.float16))),
    (ValueError, dict(history=torch.zeros(3, 9, dtype=I64))),
    (TypeError, dict(history=torch.zeros(2, 9, dtype=I32))),
    (AssertionError, dict(history=torch.zeros(9, 2, dtype=I64).t())),
    (ValueError, dict(history_lens=None)),
    (ValueError, dict(history=None, history_lens=None)),
    (TypeError, dict(history_lens=torch.zeros(2, dtype=I64))),
    (ValueError, dict(prompt_lens=torch.zeros(4, dtype=I32))),
    (TypeError, dict(repetition_penalty=torch.ones(2, dtype=torch.float64))),
    (ValueError, dict(presence_penalty=torch.ones(1))),
    (AssertionError, dict(frequency_penalty=torch.ones(4)[::2])),
    (ValueError, dict(history=None, history_lens=None, prompt_lens=None, draft_tokens=None, tree_mask=None)),
    (ValueError, dict(bias_values=None)),
    (ValueError, dict(bias_values=torch.zeros(2, 2))),
    (TypeError, dict(bias_values=torch.zeros(2, 3, dtype=BF16))),
    (ValueError, dict(allowed_mask=torch.zeros(4, 2, dtype=I32))),
    (ValueError, dict(allowed_mask=torch.zeros(2, 3, dtype=I32))),
    (TypeError, dict(allowed_mask=torch.zeros(4, 3, dtype=I64))),
    (ValueError, dict(cu_seqlens=None)),
    (ValueError, dict(cu_seqlens=torch.zeros(0, dtype=I32))),
    (ValueError, dict(draft_tokens=None)),
    (ValueError, dict(tree_mask=None)),
    (ValueError, dict(tree_mask=torch.zeros(4, 0, dtype=I64))),
    (ValueError, dict(draft_tokens=torch.zeros(3, dtype=I64))),
    (AssertionError, dict(tree_mask=torch.zeros(1, 2, dtype=I64).expand(4, 2))),
    (AssertionError, dict(allowed_mask=torch.zeros(1, 3, dtype=I32).expand(4, 3))),
    (ValueError, dict(bias_ids=torch.zeros(2, 4096, dtype=I64), bias_values=torch.zeros(2, 4096))),
    (ValueError, dict(history=torch.zeros(1, 1 << 19, dtype=I64).expand(2, 1 << 19))),
    (TypeError, dict(out=torch.zeros(4, 70, dtype=BF16))),
    (ValueError, dict(out=torch.zeros(4, 71))),
    (AssertionError, dict(out=torch.zeros(70, 4).t())),
    (AssertionError, dict(out=torch.zeros(1, 70).expand(4, 70))),
    (ValueError, dict(logits=ROWS[:4], out=ROWS[1:])),
    (ValueError, dict(logits=torch.zeros(4, 70, requires_grad=True))),
    (ValueError, dict(bias_values=torch.zeros(2, 3, requires_grad=True))),
])
def test_adjust_logits_refusals(ops, error, change):
    with pytest.raises(error):
        ops.adjust_logits(**rules(**change))


@pytest.mark.parametrize("change", [{}, dict(out=ROWS[:4], logits=ROWS[:4]), dict(draft_tokens=None, tree_mask=None), dict(prompt_lens=None), dict(logits=torch.zeros(4, 70, dtype=BF16)),
                                    dict(history=torch.zeros(1, 9, dtype=I64).expand(2, 9)), dict(allowed_mask=torch.zeros(4, 5, dtype=I32))])
def test_adjust_logits_that_fit_need_a_gpu(ops, change):
    with pytest.raises(TypeError, match="GPU"):
        ops.adjust_logits(**rules(**change))


def test_c_entries_check_their_arguments(pkg):
    from nanovllm_b200 import _abi
    lib = _abi.lib
    assert lib.b2_tree_attention_supported(32, 8, 128, 256) == 1 and lib.b2_tree_attention_supported(5, 1, 64, 48) == 1
    for bad in ((32, 7, 128, 256), (32, 8, 96, 256), (32, 8, 128, 24), (129, 1, 128, 16), (0, 1, 128, 16), (4, 0, 128, 16), (4, 2, 128, 0)):
        assert lib.b2_tree_attention_supported(*bad) == 0
    assert lib.b2_tree_attention(None, None, 0, None, None, 1, 16, None, 1, 1, None, None, None, 1, 1, 1, 1, 1, 4, 4, 128, 1.0, None, None, 0, None) == _abi.ERR_ARG
    assert lib.b2_adjust_logits(None, 8, None, 8, 0, 0, 8, _abi.LogitRules(), None) == _abi.OK
    assert lib.b2_adjust_logits(None, 8, None, 8, 0, 1, 8, _abi.LogitRules(), None) == _abi.ERR_ARG
    assert lib.b2_adjust_logits(None, 8, None, 8, 0, 1, 8, None, None) == _abi.ERR_ARG
    none = [None] * 7
    assert lib.b2_batch_inputs(None, 4, 4, None, None, 2, None, 0, None, 16, 64, 8, None, 0, 0, *none, None) == _abi.ERR_ARG
    assert lib.b2_batch_inputs(None, 4, 4, None, None, 2, None, 0, None, 0, 64, 8, None, 0, 0, *none, None) == _abi.ERR_ARG
