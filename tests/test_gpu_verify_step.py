"""A verification step of drafted trees as a serving program runs it, on a B200: inputs from the lengths, keys and values into the
cache, attention of the trees, the LM head, the rules, the pick - against the same step put together from plain statements."""
import random

import pytest
import torch

import gpu_util
import step_util as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def ops(pkg):
    gpu_util.ensure_group()
    torch.cuda.set_device(0)
    pkg.init_runtime(max_tokens=512, hidden=1024, vocab=4096, max_seqs=128)
    from nanovllm_b200 import ops
    yield ops
    pkg.shutdown_runtime()


def test_three_steps_of_a_batch(ops):
    nq, nkv, hd, bs, vocab = 8, 2, 128, 16, 4096
    g, r = torch.Generator(device=DEV).manual_seed(1), random.Random(1)
    counts = [7, 1, 16, 5]
    n, tokens = len(counts), sum(counts)

    def normal(*shape, std=1.0):
        return torch.empty(*shape, dtype=torch.bfloat16, device=DEV).normal_(0, std, generator=g)

    k_cache, v_cache = (torch.full((64, bs, nkv, hd), float("nan"), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    tables = torch.full((n, 12), -1, dtype=torch.int32, device=DEV)
    free = torch.tensor(r.sample(range(64), 64), dtype=torch.int32, device=DEV)
    num_free = torch.tensor([64], dtype=torch.int32, device=DEV)
    cached = torch.zeros(n, dtype=torch.int32, device=DEV)
    head = normal(vocab, nq * hd, std=0.05)
    history = torch.randint(0, vocab, (n, 200), generator=g, device=DEV)
    host = dict(tables=tables.tolist(), free=free.tolist(), num_free=64, cached=[0] * n)
    keys, values = [[] for _ in range(n)], [[] for _ in range(n)]  # what each request has in the cache, in order

    def step(lens, counts, mask, drafts):
        nonlocal num_free, cached
        tokens = sum(counts)
        want = ref.batch_inputs(host["tables"], host["cached"], lens, host["free"], host["num_free"], bs, 64 * bs, tokens, mask)
        got = ops.batch_inputs(tables, cached, torch.tensor(lens, dtype=torch.int32, device=DEV), free, num_free, bs, 64 * bs, tokens, None if mask is None else mask.to(DEV))
        assert [x.tolist() for x in got] == list(want[2:]) and tables.tolist() == want[0]
        host.update(tables=want[0], free=want[1], num_free=want[8][0], cached=want[7])
        q, k, v = normal(tokens, nq, hd), normal(tokens, nkv, hd), normal(tokens, nkv, hd)
        ops.store_kvcache(k, v, k_cache, v_cache, got.slot_mapping)
        at = 0
        for i, t in enumerate(counts):
            keys[i].append(k[at:at + t])
            values[i].append(v[at:at + t])
            at += t
        num_free, cached = got.num_free, got.context_lens
        if mask is None:
            return None
        o = ops.tree_attention(q, k_cache, v_cache, got.cu_seqlens_q, got.context_lens, tables, mask.to(DEV), max(counts), hd ** -0.5)
        # the plain statement over the requests' own keys and values, in rows of a cache of one block a request
        longest = max(lens)
        longest = -(-longest // 16) * 16
        pk, pv = (torch.zeros(n, longest, nkv, hd, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        for i in range(n):
            pk[i, :lens[i]], pv[i, :lens[i]] = torch.cat(keys[i]), torch.cat(values[i])
        po, size = ref.tree_attention(q, pk, pv, counts, lens, torch.arange(n, dtype=torch.int32, device=DEV).view(n, 1), mask, hd ** -0.5)
        assert ((o.double() - po).abs() <= 2.0 ** -7 * size + 2.0 ** -9 * size).all()
        logits = ops.lm_head(o.view(tokens, nq * hd), head, None)
        rules = dict(history=history, history_lens=torch.tensor([100, 0, 200, 13], dtype=torch.int32, device=DEV), prompt_lens=torch.tensor([50, 0, 10, 13], dtype=torch.int32, device=DEV),
                     repetition_penalty=torch.tensor([1.2, 1.0, 1.5, 1.1], device=DEV), presence_penalty=torch.full((n,), 0.3, device=DEV),
                     frequency_penalty=torch.full((n,), 0.1, device=DEV), cu_seqlens=got.cu_seqlens_q, draft_tokens=drafts, tree_mask=mask.to(DEV),
                     allowed_mask=torch.randint(-2 ** 31, 2 ** 31, (tokens, vocab // 32), generator=g, device=DEV).to(torch.int32))
        before = logits.clone()
        adjusted = ops.adjust_logits(logits, **rules, out=logits)
        expected = ref.adjust_logits(before.cpu(), **{k: v.cpu() for k, v in rules.items()})
        gone = torch.isinf(expected)
        assert torch.equal(torch.isinf(adjusted.cpu()), gone)
        assert ((adjusted.cpu().double() - expected).abs()[~gone] <= 2.0 ** -8 * expected.abs()[~gone] + 2.0 ** -18).all()
        picks = ops.argmax(adjusted)
        assert torch.equal(picks.cpu(), adjusted.cpu().double().argmax(-1))
        return picks

    prompts = [20, 3, 50, 33]
    step(prompts, prompts, None, None)
    lens = prompts
    for number in range(3):
        mask = ref.trees(counts, 1, number)
        drafts = torch.randint(0, vocab, (tokens,), generator=g, device=DEV)
        step([a + t for a, t in zip(lens, counts)], counts, mask, drafts)
        # the first node of each tree is kept, the others go, and with them the blocks that only they needed
        lens = [a + 1 for a in lens]
        want = ref.batch_inputs(host["tables"], host["cached"], lens, host["free"], host["num_free"], bs, 64 * bs, 0)
        got = ops.batch_inputs(tables, cached, torch.tensor(lens, dtype=torch.int32, device=DEV), free, num_free, bs, 64 * bs, 0)
        assert got.num_free.tolist() == want[8] and got.context_lens.tolist() == lens
        host.update(tables=want[0], free=want[1], num_free=want[8][0], cached=want[7])
        num_free, cached = got.num_free, got.context_lens
        for i in range(n):
            keys[i], values[i] = [torch.cat(keys[i])[:lens[i]]], [torch.cat(values[i])[:lens[i]]]


def test_a_request_that_is_not_served(ops):
    """Too few blocks for one of three requests: the others' rows are right, and its own are zero where its length is replaced by 0."""
    nq, nkv, hd, bs = 8, 2, 128, 16
    g = torch.Generator(device=DEV).manual_seed(2)

    def normal(*shape):
        return torch.empty(*shape, dtype=torch.bfloat16, device=DEV).normal_(generator=g)

    def i32(values):
        return torch.tensor(values, dtype=torch.int32, device=DEV)

    k_cache, v_cache, counts, cached = normal(8, bs, nkv, hd), normal(8, bs, nkv, hd), [4, 5, 3], [12, 14, 3]
    tables, seq_lens, mask = i32([[1, -1], [2, -1], [3, -1]]), i32([16, 19, 6]), ref.trees(counts, 1, 2)
    inp = ops.batch_inputs(tables, i32(cached), seq_lens, i32([7]), i32([0]), bs, 8 * bs, 12, mask.to(DEV))
    assert inp.context_lens.tolist() == [16, 14, 6] and inp.slot_mapping.tolist()[4:9] == [-1] * 5 and inp.cu_seqlens_q.tolist() == [0, 4, 9, 12]
    ops.store_kvcache(normal(12, nkv, hd), normal(12, nkv, hd), k_cache, v_cache, inp.slot_mapping)
    q = normal(12, nq, hd)
    lens = torch.where(inp.context_lens == seq_lens, inp.context_lens, 0)
    o = ops.tree_attention(q, k_cache, v_cache, inp.cu_seqlens_q, lens, tables, mask.to(DEV), 5, hd ** -0.5)
    want, size = ref.tree_attention(q, k_cache, v_cache, counts, [16, 0, 6], tables, mask, hd ** -0.5)
    assert (o[4:9] == 0).all() and ((o.double() - want).abs() <= 2.0 ** -7 * size + 2.0 ** -9 * size).all()
    unserved = ops.tree_attention(q, k_cache, v_cache, inp.cu_seqlens_q, inp.context_lens, tables, mask.to(DEV), 5, hd ** -0.5)
    assert torch.equal(unserved[:4], o[:4]) and torch.equal(unserved[9:], o[9:])


def test_paths_are_kept_and_the_rest_is_given_back(ops):
    """The lines between two steps: each tree's kept path moved to the places behind what was cached, then the lengths cut."""
    nkv, hd, bs, layers = 2, 128, 16, 3
    g = torch.Generator(device=DEV).manual_seed(4)
    kv_cache = torch.empty(2, layers, 16, bs, nkv, hd, dtype=torch.bfloat16, device=DEV).normal_(generator=g)
    cached, counts, paths = [14, 0, 33], [7, 3, 6], [[0, 2, 5, 6], [0], [0, 1, 4]]
    block_tables = torch.tensor([[5, -1, -1], [-1, -1, -1], [3, 9, 1]], dtype=torch.int32, device=DEV)
    free_blocks = torch.tensor([0, 2, 4, 6], dtype=torch.int32, device=DEV)
    lens, num_free = torch.tensor(cached, dtype=torch.int32, device=DEV), torch.tensor([4], dtype=torch.int32, device=DEV)
    inp = ops.batch_inputs(block_tables, lens, lens + torch.tensor(counts, dtype=torch.int32, device=DEV), free_blocks, num_free, bs, 16 * bs, sum(counts))
    old = kv_cache.clone().view(2, layers, -1, nkv, hd)
    first = torch.tensor([c for c, p in zip([0, 7, 10], paths) for _ in p], device=DEV)
    j, path = torch.tensor([i for p in paths for i in range(len(p))], device=DEV), torch.tensor([n for p in paths for n in p], device=DEV)

    dst, src = inp.slot_mapping[first + j], inp.slot_mapping[first + path]
    rows = kv_cache.view(2, layers, -1, nkv, hd)
    rows[:, :, dst] = rows[:, :, src]
    kept_lens = lens + torch.tensor([len(p) for p in paths], dtype=torch.int32, device=DEV)
    kept = ops.batch_inputs(block_tables, inp.context_lens, kept_lens, free_blocks, inp.num_free, bs, 16 * bs, 0)

    assert kept.context_lens.tolist() == [18, 1, 36] and kept.num_free.tolist() == [2] and block_tables[:, 0].tolist()[0] == 5
    tables = block_tables.tolist()
    for i, (c, p) in enumerate(zip(cached, paths)):
        def slot(place):
            return tables[i][place // bs] * bs + place % bs
        for place in range(c):
            assert torch.equal(rows[:, :, slot(place)], old[:, :, slot(place)])
        for k, node in enumerate(p):
            assert torch.equal(rows[:, :, slot(c + k)], old[:, :, slot(c + node)]), (i, k)
