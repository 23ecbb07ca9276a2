"""Decode attention straight behind the kernel that makes its lengths and tables, on a B200: it reads them ahead of its dependency wait, so
the kernel before it must not have let it in until they are there.  Results equal bit for bit to those of the same calls with a
synchronisation between them, and those are held against the definition in 64 bits."""
import random

import pytest
import torch

import step_util as ref
from tests.gpu_util import ensure_group

pytestmark = pytest.mark.gpu
DEV = "cuda"
BS, BLOCKS, NQ, NKV, HD = 64, 2000, 4, 2, 128


@pytest.fixture(scope="module")
def ops(pkg):
    ensure_group()
    from nanovllm_b200 import ops
    from nanovllm_b200.runtime import init_runtime, shutdown_runtime
    init_runtime(max_tokens=1024, hidden=1024)
    yield ops
    shutdown_runtime()


@pytest.fixture(scope="module")
def cache(ops):
    g = torch.Generator(device=DEV).manual_seed(3)
    return tuple(torch.empty(BLOCKS, BS, NKV, HD, dtype=torch.bfloat16, device=DEV).normal_(generator=g) for _ in range(2))


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def queries(n, seed):
    return torch.empty(n, NQ, HD, dtype=torch.bfloat16, device=DEV).normal_(generator=torch.Generator(device=DEV).manual_seed(seed))


def hold_against_definition(o, q, cache, lens, tables):
    """Products and sums of 128 terms in 32 bits are below the roundings: of the probabilities and of the result, 2^-8 each (the
    rounded probabilities' sum included, one more), of the terms' sizes."""
    ones = torch.full((len(lens), 1), 1, dtype=torch.int64)
    want, size = ref.tree_attention(q, *cache, [1 if n else 0 for n in lens], lens, tables, ones, HD ** -0.5)
    assert ((o.double() - want).abs() <= 3 * 2.0 ** -8 * size + 1e-6).all()


@pytest.mark.parametrize("store", [False, True])
@pytest.mark.parametrize("n", [1, 40, 512])
def test_decode_attention_behind_batch_inputs(ops, cache, n, store):
    """Every context is at a block's end or has none, so that each row's last tile is in a block that this very step has opened."""
    r = random.Random(n)
    cached = [r.choice((0, BS, 2 * BS)) for _ in range(n)]
    free = r.sample(range(1, BLOCKS), BLOCKS - 1)
    tables = [[free.pop() for _ in range(c // BS)] + [-1] * (4 - c // BS) for c in cached]
    wanted = [c + 1 for c in cached]
    q, key, value = queries(n, 1), queries(n, 2)[:, :NKV], queries(n, 3)[:, :NKV]
    key, value = key.contiguous(), value.contiguous()
    t, f, stack = i32(tables), i32(free), i32(free)
    c, w, height = i32(cached), i32(wanted), i32([len(free)])

    def step(wait):
        inp = ops.batch_inputs(t, c, w, f, height, BS, BLOCKS * BS, n)
        if wait:
            torch.cuda.synchronize()
        if store:
            ops.store_kvcache(key, value, *cache, inp.slot_mapping)
        if wait:
            torch.cuda.synchronize()
        return inp, ops.paged_attention(q, *cache, inp.context_lens, t, HD ** -0.5)

    inp, want = step(wait=True)
    assert inp.context_lens.tolist() == wanted
    hold_against_definition(want, q, cache, wanted, t)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, got = step(wait=False)
    torch.cuda.synchronize()
    for i in range(50):
        # another deal of the blocks each time, and tables that lack the new ones before the step
        r.shuffle(free)
        f.copy_(i32(free))
        t.copy_(i32(tables))
        _, want = step(wait=True)
        f.copy_(i32(free))
        t.copy_(i32(tables))
        graph.replay()
        assert torch.equal(got, want), f"replay {i}"
        f.copy_(i32(free))
        t.copy_(i32(tables))
        _, eager = step(wait=False)
        assert torch.equal(eager, want), f"call {i}"


@pytest.mark.parametrize("n", [1, 33, 128, 500])
def test_decode_attention_behind_advance_decode(ops, cache, n):
    """Contexts on both sides of a block's end; the last row of each warp is frozen, so that its threads have less to do than the others."""
    r = random.Random(n)
    lens = [r.choice((1, 31, BS - 1, BS, BS + 1, 2 * BS - 1)) for _ in range(n)]
    blocks = r.sample(range(BLOCKS), 3 * n)
    t = i32(blocks).view(n, 3)
    q = queries(n, 4)
    tokens, ids = torch.arange(n, device=DEV), torch.zeros(n, dtype=torch.int64, device=DEV)
    start = i32(lens)
    slot = i32([-1 if i % 32 == 31 else blocks[3 * i + (x - 1) // BS] * BS + (x - 1) % BS for i, x in enumerate(lens)])
    position, c, s = torch.zeros(n, dtype=torch.int64, device=DEV), torch.zeros_like(start), torch.zeros_like(slot)

    def reset():
        position.copy_(start - 1)
        c.copy_(start)
        s.copy_(slot)

    def step(wait):
        ops.advance_decode(tokens, ids, position, c, s, t, BS, BLOCKS * BS)
        if wait:
            torch.cuda.synchronize()
        return ops.paged_attention(q, *cache, c, t, HD ** -0.5)

    reset()
    want = step(wait=True)
    after = [x + (i % 32 != 31) for i, x in enumerate(lens)]
    assert c.tolist() == after
    hold_against_definition(want, q, cache, after, t)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(wait=False)
    for i in range(50):
        reset()
        graph.replay()
        assert torch.equal(got, want), f"replay {i}"
        reset()
        assert torch.equal(step(wait=False), want), f"call {i}"


@pytest.mark.parametrize("n, heads", [(40, (4, 2)), (512, (4, 2)), (300, (8, 2))])
def test_steps_one_after_the_other(ops, cache, n, heads):
    """Eight steps back to back, each of which changes lengths and tables that the attention before it has read: nothing of the step before is seen."""
    r = random.Random(n)
    cached = [r.choice((0, 1, BS - 5, BS - 1, BS)) for _ in range(n)]
    free = r.sample(range(1, BLOCKS), BLOCKS - 1)
    tables = [[free.pop() for _ in range(-(-c // BS))] + [-1] * (3 - -(-c // BS)) for c in cached]
    q = torch.empty(n, heads[0], HD, dtype=torch.bfloat16, device=DEV).normal_(generator=torch.Generator(device=DEV).manual_seed(5))
    t, f, height, start = i32(tables), i32(free), i32([len(free)]), i32(cached)
    wanted = [start + r.choice((3, 5)) * (i + 1) for i in range(8)]

    def steps(wait):
        lens, left, out = start, height, []
        for w in wanted:
            inp = ops.batch_inputs(t, lens, w, f, left, BS, BLOCKS * BS, 5 * n)
            if wait:
                torch.cuda.synchronize()
            out.append(ops.paged_attention(q, *cache, inp.context_lens, t, HD ** -0.5))
            if wait:
                torch.cuda.synchronize()
            lens, left = inp.context_lens, inp.num_free
        return torch.stack(out)

    def reset():
        t.copy_(i32(tables))
        f.copy_(i32(free))

    want = steps(wait=True)
    assert len({x.sum().item() for x in want.double()}) == 8
    reset()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = steps(wait=False)
    for i in range(30):
        reset()
        graph.replay()
        assert torch.equal(got, want), f"replay {i}"
