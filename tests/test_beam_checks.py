"""What the operators of a beam-search step refuse, on tensors that never reach a GPU: every refusal is an error before anything is launched, and a call
that fits gets as far as the check for the GPU."""
import ctypes as C

import pytest
import torch

I32, I64, F32, BF16 = torch.int32, torch.int64, torch.float32, torch.bfloat16


def zeros(*shape, dtype=I32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.fixture
def ops(pkg, monkeypatch):
    from nanovllm_b200 import ops

    class Runtime:
        handle = None

    monkeypatch.setattr(ops, "get_runtime", lambda: Runtime)
    return ops


def prefix_args(**kw):
    a = dict(q=zeros(5, 4, 128, dtype=BF16), k_cache=zeros(3, 16, 2, 128, dtype=BF16), v_cache=zeros(3, 16, 2, 128, dtype=BF16), cu_groups=zeros(3), prefix_lens=zeros(2), context_lens=zeros(5),
             block_tables=zeros(5, 2), max_group=3, scale=0.1)
    a.update(kw)
    return a


@pytest.mark.parametrize("error, change", [
    (ValueError, dict(q=zeros(5, 512, dtype=BF16))),
    (TypeError, dict(q=zeros(5, 4, 128, dtype=F32))),
    (ValueError, dict(q=zeros(5, 3, 128, dtype=BF16))),
    (ValueError, dict(q=zeros(5, 4, 64, dtype=BF16))),
    (ValueError, dict(q=zeros(5, 4, 96, dtype=BF16), k_cache=zeros(3, 16, 2, 96, dtype=BF16), v_cache=zeros(3, 16, 2, 96, dtype=BF16))),
    (ValueError, dict(q=zeros(5, 258, 128, dtype=BF16))),
    (ValueError, dict(k_cache=zeros(3, 24, 2, 128, dtype=BF16), v_cache=zeros(3, 24, 2, 128, dtype=BF16))),
    (ValueError, dict(k_cache=zeros(48, 2, 128, dtype=BF16))),
    (TypeError, dict(k_cache=zeros(3, 16, 2, 128, dtype=F32))),
    (ValueError, dict(v_cache=zeros(2, 16, 2, 128, dtype=BF16))),
    (TypeError, dict(v_cache=zeros(3, 16, 2, 128, dtype=F32))),
    (AssertionError, dict(k_cache=zeros(3, 2, 16, 128, dtype=BF16).transpose(1, 2))),
    (AssertionError, dict(q=zeros(5, 128, 4, dtype=BF16).transpose(1, 2))),
    (AssertionError, dict(q=zeros(5, 4, 129, dtype=BF16)[:, :, :128])),
    (ValueError, dict(cu_groups=zeros(2))),
    (TypeError, dict(cu_groups=zeros(3, dtype=I64))),
    (TypeError, dict(prefix_lens=zeros(2, dtype=I64))),
    (AssertionError, dict(prefix_lens=zeros(4)[::2])),
    (ValueError, dict(context_lens=zeros(4))),
    (TypeError, dict(context_lens=zeros(5, dtype=F32))),
    (ValueError, dict(block_tables=zeros(4, 2))),
    (ValueError, dict(block_tables=zeros(5, 0))),
    (TypeError, dict(block_tables=zeros(5, 2, dtype=I64))),
    (AssertionError, dict(block_tables=zeros(1, 2).expand(5, 2))),
    (AssertionError, dict(block_tables=zeros(2, 5).t())),
    (ValueError, dict(max_group=-1)),
    (ValueError, dict(max_group=0)),
    (ValueError, dict(q=zeros(1025, 4, 128, dtype=BF16), context_lens=zeros(1025), block_tables=zeros(1025, 2))),
    (ValueError, dict(cu_groups=zeros(514), prefix_lens=zeros(513))),
    (ValueError, dict(block_tables=zeros(1, 1 << 23).expand(5, 1 << 23))),
    (ValueError, dict(q=torch.zeros(5, 4, 128, dtype=BF16, requires_grad=True))),
])
def test_shared_prefix_attention_refusals(ops, error, change):
    with pytest.raises(error):
        ops.shared_prefix_attention(**prefix_args(**change))


@pytest.mark.parametrize("change", [{}, dict(q=zeros(5, 6, 4, 128, dtype=BF16)[:, 2]), dict(block_tables=zeros(5, 7)[:, 3:5]), dict(cu_groups=zeros(1), prefix_lens=zeros(0), max_group=0),
                                    dict(q=zeros(0, 4, 128, dtype=BF16), context_lens=zeros(0), block_tables=zeros(0, 2)), dict(q=zeros(5, 256, 128, dtype=BF16)), dict(max_group=10 ** 6)])
def test_shared_prefix_attention_calls_that_fit_need_a_gpu(ops, change):
    with pytest.raises(TypeError, match="GPU"):
        ops.shared_prefix_attention(**prefix_args(**change))


def select_args(**kw):
    a = dict(logits=zeros(6, 11, dtype=BF16), scores=zeros(2, 3, dtype=F32), picks=4, finished=None, eos_token=None)
    a.update(kw)
    return a


@pytest.mark.parametrize("error, change", [
    (ValueError, dict(scores=zeros(6, dtype=F32))),
    (TypeError, dict(scores=zeros(2, 3, dtype=torch.float64))),
    (AssertionError, dict(scores=zeros(3, 2, dtype=F32).t())),
    (ValueError, dict(logits=zeros(66, dtype=BF16))),
    (TypeError, dict(logits=zeros(6, 11, dtype=torch.float16))),
    (ValueError, dict(logits=zeros(5, 11, dtype=BF16))),
    (ValueError, dict(logits=zeros(6, 0, dtype=BF16))),
    (ValueError, dict(picks=0)),
    (ValueError, dict(picks=65)),
    (ValueError, dict(logits=zeros(33, 11, dtype=BF16), scores=zeros(1, 33, dtype=F32))),
    (ValueError, dict(logits=zeros(0, 11, dtype=BF16), scores=zeros(2, 0, dtype=F32), picks=1)),
    (TypeError, dict(finished=zeros(2, 3, dtype=torch.uint8))),
    (ValueError, dict(finished=zeros(2, 4, dtype=torch.bool))),
    (AssertionError, dict(finished=zeros(3, 2, dtype=torch.bool).t())),
    (ValueError, dict(eos_token=-2)),
    (ValueError, dict(eos_token=1 << 40)),
    (ValueError, dict(logits=torch.zeros(6, 11, dtype=BF16, requires_grad=True))),
    (ValueError, dict(scores=torch.zeros(2, 3, requires_grad=True))),
])
def test_beam_select_refusals(ops, error, change):
    with pytest.raises(error):
        ops.beam_select(**select_args(**change))


@pytest.mark.parametrize("change", [{}, dict(picks=None), dict(picks=64), dict(logits=zeros(6, 11, dtype=F32)), dict(logits=zeros(11, 6, dtype=BF16).t()), dict(finished=zeros(2, 3, dtype=torch.bool)),
                                    dict(eos_token=10), dict(eos_token=500), dict(logits=zeros(0, 11, dtype=BF16), scores=zeros(0, 3, dtype=F32))])
def test_beam_select_calls_that_fit_need_a_gpu(ops, change):
    with pytest.raises(TypeError, match="GPU"):
        ops.beam_select(**select_args(**change))


def reorder_args(**kw):
    a = dict(parents=zeros(2, 3), block_tables=zeros(6, 4), context_lens=zeros(6), free_blocks=zeros(9), num_free=zeros(1), kv_cache=zeros(2, 3, 7, 16, 2, 64, dtype=BF16), first_blocks=None,
             history=zeros(6, 20, dtype=I64), history_lens=zeros(6), tokens=zeros(2, 3, dtype=I64))
    a.update(kw)
    return a


STACK = zeros(40)
CACHE = zeros(2, 7, 16, 2, 64, dtype=BF16)


@pytest.mark.parametrize("error, change", [
    (ValueError, dict(parents=zeros(6))),
    (TypeError, dict(parents=zeros(2, 3, dtype=I64))),
    (AssertionError, dict(parents=zeros(3, 2).t())),
    (ValueError, dict(parents=zeros(1, 33), block_tables=zeros(33, 4), context_lens=zeros(33), history=None, history_lens=None, tokens=None)),
    (ValueError, dict(parents=zeros(257, 32), block_tables=zeros(8224, 1), context_lens=zeros(8224), history=None, history_lens=None, tokens=None)),
    (ValueError, dict(block_tables=zeros(5, 4))),
    (ValueError, dict(block_tables=zeros(6, 0))),
    (TypeError, dict(block_tables=zeros(6, 4, dtype=I64))),
    (AssertionError, dict(block_tables=zeros(1, 4).expand(6, 4))),
    (ValueError, dict(context_lens=zeros(5))),
    (TypeError, dict(context_lens=zeros(6, dtype=I64))),
    (AssertionError, dict(free_blocks=zeros(18)[::2])),
    (TypeError, dict(free_blocks=zeros(9, dtype=I64))),
    (ValueError, dict(num_free=zeros(2))),
    (ValueError, dict(first_blocks=zeros(3))),
    (TypeError, dict(first_blocks=zeros(2, dtype=I64))),
    (ValueError, dict(kv_cache=zeros(7, 16, 64, dtype=BF16))),
    (ValueError, dict(kv_cache=zeros(2, 0, 16, 2, 64, dtype=BF16))),
    (AssertionError, dict(kv_cache=zeros(2, 7, 2, 16, 64, dtype=BF16).transpose(2, 3))),
    (AssertionError, dict(kv_cache=zeros(2, 7, 16, 1, 4, dtype=BF16))),
    (AssertionError, dict(kv_cache=zeros(1 + 2 * 7 * 16 * 8, dtype=BF16)[1:].view(2, 7, 16, 1, 8))),
    (AssertionError, dict(kv_cache=CACHE[:1].expand(2, 7, 16, 2, 64))),
    (AssertionError, dict(kv_cache=zeros(3, 4, 7, 16, 2, 64, dtype=BF16)[:, :3])),
    (ValueError, dict(history=None)),
    (ValueError, dict(history_lens=None)),
    (ValueError, dict(history=None, history_lens=None)),
    (ValueError, dict(history=zeros(5, 20, dtype=I64))),
    (TypeError, dict(history=zeros(6, 20))),
    (AssertionError, dict(history=zeros(1, 20, dtype=I64).expand(6, 20))),
    (TypeError, dict(history_lens=zeros(6, dtype=I64))),
    (ValueError, dict(tokens=zeros(6, dtype=I64))),
    (TypeError, dict(tokens=zeros(2, 3))),
    (ValueError, dict(free_blocks=STACK[:9], block_tables=STACK[8:32].view(6, 4))),
    (ValueError, dict(free_blocks=STACK[:9], num_free=STACK[8:9])),
    (ValueError, dict(free_blocks=STACK[:9], parents=STACK[3:9].view(2, 3))),
    (ValueError, dict(kv_cache=CACHE, history=CACHE.view(-1).view(I64)[:120].view(6, 20))),
    (ValueError, dict(kv_cache=CACHE, free_blocks=CACHE.view(-1).view(I32)[:9])),
    (ValueError, dict(parents=zeros(1, 1), block_tables=torch.empty(1, 1 << 28, dtype=I32), context_lens=zeros(1), history=None, history_lens=None, tokens=None)),
    (ValueError, dict(kv_cache=torch.zeros(2, 7, 16, 2, 64, dtype=BF16, requires_grad=True))),
])
def test_reorder_beams_refusals(ops, error, change):
    with pytest.raises(error):
        ops.reorder_beams(**reorder_args(**change))


@pytest.mark.parametrize("change", [{}, dict(first_blocks=zeros(2)), dict(history=None, history_lens=None, tokens=None), dict(tokens=None), dict(kv_cache=CACHE[0]), dict(kv_cache=zeros(0, 7, 16, 2, 64, dtype=BF16)),
                                    dict(kv_cache=zeros(2, 9, 16, 2, 64, dtype=BF16)[:, :7]), dict(history=zeros(6, 0, dtype=I64)), dict(free_blocks=zeros(0)), dict(block_tables=zeros(6, 9)[:, 2:6]),
                                    dict(parents=zeros(0, 3), block_tables=zeros(0, 4), context_lens=zeros(0), history=None, history_lens=None, tokens=None)])
def test_reorder_beams_calls_that_fit_need_a_gpu(ops, change):
    with pytest.raises(TypeError, match="GPU"):
        ops.reorder_beams(**reorder_args(**change))


def test_workspaces_and_bad_arguments_of_the_c_entries(pkg):
    """Shapes that are not served have no workspace; a call without a context is an error, not a launch."""
    from nanovllm_b200 import _abi
    lib = _abi.lib
    for nq, nkv, hd, bs, served in ((4, 2, 128, 16, 1), (128, 1, 64, 48, 1), (129, 1, 64, 16, 0), (4, 3, 128, 16, 0), (4, 2, 96, 16, 0), (4, 2, 128, 8, 0), (0, 1, 64, 16, 0), (4, 0, 64, 16, 0), (4, -2, 64, 16, 0),
                                    (4, 2, 128, 0, 0), (4, 2, 128, -16, 0)):
        assert lib.b2_prefix_attention_supported(nq, nkv, hd, bs) == served
    assert lib.b2_prefix_attention_workspace(None, 4, 1, 4, 2, 128, 16, 9) == -1
    assert lib.b2_beam_select_workspace(None, 1, 1, 10, 1, 0) == -1
    assert lib.b2_reorder_beams_workspace(2, 4, 10) >= 8 * 10 * 4
    assert lib.b2_reorder_beams_workspace(0, 4, 10) == 0
    for n, beams, width in ((-1, 4, 10), (2, 0, 10), (2, 33, 10), (257, 32, 10), (2, 4, -1)):
        assert lib.b2_reorder_beams_workspace(n, beams, width) == -1
    assert lib.b2_prefix_attention(None, None, 512, None, None, 3, 16, None, 2, 2, None, None, None, 1, 3, 5, 4, 2, 128, C.c_float(0.1), None, None, 0, None) != 0
    assert lib.b2_beam_select(None, None, 11, 0, 2, 3, 11, None, None, 4, -1, None, None, None, None, None, 0, None) != 0
    assert lib.b2_reorder_beams(None, None, 2, 3, None, 4, 4, None, None, None, 9, None, 16, None, 2, 0, 7, 256, None, 0, 0, None, None, None, None, None, None, None, None, 0, None) != 0
