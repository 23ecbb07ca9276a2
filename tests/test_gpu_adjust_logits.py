"""ops.adjust_logits on a B200 against its definition in 64 bits.

Tolerance, per element: four operations in 32 bits (quotient or product, product with the count, two differences, a sum), each off by at most
2^-24 of its result, whose sizes are below |x| max(r, 1 / r) + frequency count + presence + |bias| =: size; so 5 * 2^-24 size, and for bf16 logits
the rounding at the end, 2^-8 of the result.  Elements that no rule touches are equal bit for bit."""
import random

import pytest
import torch

import step_util as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def ops(pkg):
    from nanovllm_b200 import ops
    return ops


def request(n, vocab, rows, seed, history=40, bias=5, mask=True, penalties=True, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    r = random.Random(seed)
    a = {}
    if penalties:
        a["history"] = torch.randint(-2, min(vocab, 50) + 1, (n, history), generator=g)
        a["history"][:, ::7] = vocab - 1
        a["history_lens"] = torch.tensor([r.randint(0, history) for _ in range(n)], dtype=torch.int32)
        a["prompt_lens"] = torch.tensor([r.randint(0, int(x)) for x in a["history_lens"]], dtype=torch.int32)
        a["repetition_penalty"] = torch.tensor([r.choice((1.0, 1.3, 0.7)) for _ in range(n)])
        a["presence_penalty"] = torch.tensor([r.choice((0.0, 0.9, -0.4)) for _ in range(n)])
        a["frequency_penalty"] = torch.tensor([r.choice((0.0, 0.21, -0.3)) for _ in range(n)])
    if bias:
        a["bias_ids"] = torch.randint(-2, vocab + 2, (n, bias), generator=g)
        a["bias_ids"][:, -1] = a["bias_ids"][:, 0]  # the last of equal ids counts
        a["bias_values"] = torch.randn(n, bias, generator=g) * 4
    if mask:
        a["allowed_mask"] = torch.randint(-2 ** 31, 2 ** 31, (rows, -(-vocab // 32)), generator=g).to(torch.int32)
    logits = (torch.randn(rows, vocab, generator=g) * 3).to(dtype)
    return logits, a


def on_gpu(a):
    return {k: v.to(DEV) for k, v in a.items()}


def check(got, logits, a, what=""):
    want = ref.adjust_logits(logits, **a)
    got, dtype = got.cpu(), logits.dtype
    assert got.dtype == dtype and got.shape == logits.shape
    untouched = want == logits.double()
    assert torch.equal(got[untouched].double(), logits[untouched].double()), what
    gone = torch.isinf(want)
    assert torch.equal(got[gone].double(), want[gone]), what
    x = logits.double().abs()
    size = x.clone()
    if "repetition_penalty" in a:
        r = a["repetition_penalty"].double()
        size = size * torch.maximum(r, 1 / r).max()
        size = size + a["frequency_penalty"].double().abs().max() * (a["history"].shape[1] + 64) + a["presence_penalty"].double().abs().max()
    if "bias_values" in a:
        size = size + a["bias_values"].double().abs().max()
    half = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    bound = 5 * 2.0 ** -24 * size * (1 + half) + half * want.abs()
    err = (got.double() - want).abs()
    fine = ~gone
    assert (err[fine] <= bound[fine]).all(), f"{what}: off by {(err[fine] - bound[fine]).max().item():.3e} more than the bound"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 31, 33, 1000, 8191, 8192, 8193, 8200, 20001])
def test_vocabularies(ops, vocab, dtype):
    logits, a = request(3, vocab, 3, seed=vocab, dtype=dtype)
    check(ops.adjust_logits(logits.to(DEV), **on_gpu(a)), logits, a)


@pytest.mark.parametrize("leave", ["penalties", "bias", "mask", "all"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rules_left_out(ops, leave, dtype):
    logits, a = request(4, 9001, 4, seed=2, penalties=leave not in ("penalties", "all"), bias=0 if leave in ("bias", "all") else 6, mask=leave not in ("mask", "all"), dtype=dtype)
    got = ops.adjust_logits(logits.to(DEV), **on_gpu(a))
    check(got, logits, a)
    if leave == "all":
        assert torch.equal(got.cpu(), logits)


@pytest.mark.parametrize("name", ["repetition_penalty", "presence_penalty", "frequency_penalty", "prompt_lens"])
def test_one_of_the_penalties_left_out(ops, name):
    logits, a = request(4, 3001, 4, seed=3)
    b = dict(a)
    del b[name]
    got = ops.adjust_logits(logits.to(DEV), **on_gpu(b))
    want = ref.adjust_logits(logits, **b)
    gone = torch.isinf(want)
    assert torch.equal(torch.isinf(got.cpu()), gone)
    assert ((got.cpu().double() - want)[~gone].abs() <= 2.0 ** -20 * 64).all()


@pytest.mark.parametrize("history", [1, 100, 5000])
def test_long_histories_of_few_tokens(ops, history):
    """Thousands of occurrences of one token are counted exactly."""
    logits, a = request(2, 40000, 2, seed=4, history=history)
    a["history"][0] = 17
    a["history_lens"][:] = history
    a["prompt_lens"][:] = history // 3
    check(ops.adjust_logits(logits.to(DEV), **on_gpu(a)), logits, a)


def test_lengths_outside_the_history(ops):
    logits, a = request(4, 500, 4, seed=5)
    a["history_lens"] = torch.tensor([-3, 0, 41, 2 ** 31 - 1], dtype=torch.int32)
    a["prompt_lens"] = torch.tensor([-1, 5, 60, 2], dtype=torch.int32)
    check(ops.adjust_logits(logits.to(DEV), **on_gpu(a)), logits, a)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_trees(ops, dtype):
    counts = [5, 0, 70, 1, 12]
    rows = sum(counts) + 3
    logits, a = request(5, 9000, rows, seed=6, dtype=dtype)
    a["cu_seqlens"] = ref.cumulative(counts)
    a["draft_tokens"] = torch.randint(0, 30, (rows,), generator=torch.Generator().manual_seed(6))
    a["draft_tokens"][3], a["draft_tokens"][9] = -1, 9000
    a["tree_mask"] = torch.cat([ref.trees(counts, 2, 6), torch.full((3, 2), -1, dtype=torch.int64)])
    got = ops.adjust_logits(logits.to(DEV), **on_gpu(a))
    check(got, logits, a)
    assert torch.equal(got[-3:].cpu(), logits[-3:])  # rows behind the last request
    x = logits.to(DEV)
    ops.adjust_logits(x, **on_gpu(a), out=x)
    assert torch.equal(x, got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_several_rows_of_a_request_without_drafts(ops, dtype):
    counts = [5, 0, 70, 1, 12]
    rows = sum(counts) + 3
    logits, a = request(5, 9000, rows, seed=16, dtype=dtype)
    a["cu_seqlens"] = ref.cumulative(counts)
    check(ops.adjust_logits(logits.to(DEV), **on_gpu(a)), logits, a)


def test_trees_over_several_slices_between_rows_without_a_path(ops):
    """Rows with and without a path by turns, an odd number of them, more steps than CTAs."""
    counts = [1, 2, 0, 3, 5, 1, 1]
    rows = sum(counts)
    logits, a = request(7, 60001, rows, seed=18, dtype=torch.bfloat16)
    logits, a["allowed_mask"] = logits.repeat(40, 1), a["allowed_mask"].repeat(40, 1)
    a = {k: v if k == "allowed_mask" else v.repeat(40, *[1] * (v.dim() - 1)) for k, v in a.items()}
    a["cu_seqlens"] = ref.cumulative(counts * 40)
    a["draft_tokens"] = torch.randint(0, 40, (rows * 40,), generator=torch.Generator().manual_seed(18))
    a["tree_mask"] = ref.trees(counts * 40, 1, 18)
    a["tree_mask"][::3] = 0
    got = ops.adjust_logits(logits.to(DEV), **on_gpu(a))
    check(got, logits, a)


def test_trees_without_a_history(ops):
    counts = [4, 9]
    logits, a = request(2, 500, 13, seed=7, penalties=False)
    a.update(repetition_penalty=torch.tensor([1.5, 2.0]), presence_penalty=torch.tensor([0.25, 0.5]), frequency_penalty=torch.tensor([0.5, 0.25]), cu_seqlens=ref.cumulative(counts),
             draft_tokens=torch.randint(0, 5, (13,), generator=torch.Generator().manual_seed(7)), tree_mask=ref.trees(counts, 1, 7))
    want = ref.adjust_logits(logits, **a)
    got = ops.adjust_logits(logits.to(DEV), **on_gpu(a)).cpu()
    gone = torch.isinf(want)
    assert torch.equal(torch.isinf(got), gone) and ((got.double() - want)[~gone].abs() <= 2.0 ** -20 * 64).all()


def test_many_rows_of_a_request(ops):
    """More rows than CTAs: rows of a request share the counts of its history."""
    counts = [300, 2, 333]
    rows = sum(counts)
    logits, a = request(3, 10000, rows, seed=8, bias=3, mask=False, dtype=torch.bfloat16)
    a["cu_seqlens"] = ref.cumulative(counts)
    a["draft_tokens"] = torch.randint(0, 40, (rows,), generator=torch.Generator().manual_seed(8))
    a["tree_mask"] = ref.trees(counts, 6, 8)
    check(ops.adjust_logits(logits.to(DEV), **on_gpu(a)), logits, a)


def test_a_list_longer_than_a_block(ops):
    """Every token of a slice in the history, and paths of more nodes than a block has threads."""
    rows = 700
    logits, a = request(1, 9000, rows, seed=17, history=9000, bias=40, dtype=torch.bfloat16)
    a["history"][0] = torch.randperm(9000, generator=torch.Generator().manual_seed(17))
    a["history_lens"][:], a["prompt_lens"][:] = 9000, 4000
    a["cu_seqlens"] = ref.cumulative([rows])
    a["draft_tokens"] = torch.randint(0, 200, (rows,), generator=torch.Generator().manual_seed(17))
    a["tree_mask"] = ref.masks([(2 << i) - 1 for i in range(rows)], 11)
    keep = [0, 1, 300, 699]
    b = on_gpu(a)
    got = ops.adjust_logits(logits.to(DEV), **b)
    x = logits.to(DEV)
    ops.adjust_logits(x, **b, out=x)
    assert torch.equal(x, got)
    # (the definition a few rows at a time: a row's path as the end of a longer history)
    for row in keep:
        one = dict(a, history=torch.cat([a["history"], a["draft_tokens"][:row + 1].view(1, -1)], 1), history_lens=torch.tensor([9000 + row + 1], dtype=torch.int32),
                   allowed_mask=a["allowed_mask"][row:row + 1])
        for name in ("cu_seqlens", "draft_tokens", "tree_mask"):
            del one[name]
        check(got[row:row + 1], logits[row:row + 1], one, f"row {row}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_in_place_and_into_another_tensor(ops, dtype):
    logits, a = request(5, 8300, 5, seed=9, dtype=dtype)
    b = on_gpu(a)
    want = ops.adjust_logits(logits.to(DEV), **b)
    x = logits.to(DEV)
    assert ops.adjust_logits(x, **b, out=x) is not None and torch.equal(x, want)
    big = torch.full((5, 9000), 7.0, dtype=dtype, device=DEV)
    for first in (0, 1, 3, 8):
        big.fill_(7)
        out = big[:, first:first + 8300]
        ops.adjust_logits(logits.to(DEV), **b, out=out)
        assert torch.equal(out, want) and (big[:, :first] == 7).all() and (big[:, first + 8300:] == 7).all()
        wide = torch.zeros(5, 9001, dtype=dtype, device=DEV)
        wide[:, first:first + 8300] = logits.to(DEV)
        x = wide[:, first:first + 8300]
        assert torch.equal(ops.adjust_logits(x, **b), want)
        ops.adjust_logits(x, **b, out=x)
        assert torch.equal(x, want) and not wide[:, first + 8300:].any()


def test_transposed_logits_and_a_shared_history(ops):
    logits, a = request(4, 600, 4, seed=10)
    a["history"] = a["history"][:1].expand(4, -1)
    a["bias_ids"], a["bias_values"] = a["bias_ids"][:1].expand(4, -1), a["bias_values"][:1].expand(4, -1)
    b = on_gpu(a)
    b["history"] = b["history"][:1].contiguous().expand(4, -1)
    check(ops.adjust_logits(logits.t().contiguous().to(DEV).t(), **b), logits, a)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_infinities_and_nan(ops, dtype):
    """Forbidden tokens are -inf whatever they were; -inf stays -inf under penalties; untouched NaN stay."""
    logits, a = request(2, 640, 2, seed=11, dtype=dtype)
    logits[:, ::5], logits[:, 1::5], logits[:, 2::50], logits[:, 3::50] = float("nan"), -float("inf"), torch.finfo(dtype).min, torch.finfo(dtype).max
    a["repetition_penalty"][:] = 1.0
    got = ops.adjust_logits(logits.to(DEV), **on_gpu(a)).cpu()
    words = a["allowed_mask"].long() & 0xffffffff
    k = torch.arange(640)
    allowed = ((words[:, k // 32] >> (k % 32)) & 1).bool()
    assert torch.equal(got == -float("inf"), ~allowed | (logits == -float("inf")))
    assert torch.equal(torch.isnan(got), allowed & torch.isnan(logits))


def test_a_mask_that_leaves_nothing(ops):
    logits, a = request(2, 640, 2, seed=12)
    a["allowed_mask"][1] = 0
    got = ops.adjust_logits(logits.to(DEV), **on_gpu(a)).cpu()
    assert (got[1] == -float("inf")).all() and not (got[0] == -float("inf")).all()


def test_no_rows(ops):
    logits, a = request(3, 640, 3, seed=13)
    a = {k: v[:0] for k, v in on_gpu(a).items()}
    assert ops.adjust_logits(logits[:0].to(DEV), **a).shape == (0, 640)


def test_captured_and_on_another_stream(ops):
    logits, a = request(6, 30000, 6, seed=14, dtype=torch.bfloat16)
    x, b = logits.to(DEV), on_gpu(a)
    ops.adjust_logits(x, **b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.adjust_logits(x, **b)
    other, c = request(6, 30000, 6, seed=15, dtype=torch.bfloat16)
    x.copy_(other)
    for k in b:
        b[k].copy_(c[k])
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        graph.replay()
        eager = ops.adjust_logits(x, **b)
    stream.synchronize()
    check(out, other, c)
    assert torch.equal(out, eager)


@pytest.mark.parametrize("rules", ["all", "mask", "trees"])
@pytest.mark.parametrize("first", [1, 5])
def test_rows_before_the_first_request_are_copied(ops, first, rules):
    """cu_seqlens need not begin at 0: the rows before its first element belong to nobody, like those behind its last, in every slice of the vocabulary."""
    cu = torch.tensor([first, first, first + 3, first + 4], dtype=torch.int32)
    rows = first + 6
    logits, a = request(3, 9001, rows, seed=first, penalties=rules != "mask", bias=0 if rules == "mask" else 4)
    a["cu_seqlens"] = cu
    if rules == "trees":
        a["draft_tokens"] = torch.arange(rows) * 700
        a["tree_mask"] = torch.full((rows, 1), -1, dtype=torch.int64)
    got = ops.adjust_logits(logits.to(DEV), **on_gpu(a))
    check(got, logits, a)
    assert torch.equal(got[:first].cpu(), logits[:first]) and torch.equal(got[first + 4:].cpu(), logits[first + 4:])
    assert not torch.equal(got[first:first + 4].cpu(), logits[first:first + 4])
