"""ops.batch_inputs on a B200 against the requests taken one after the other on the host: whole numbers, equal."""
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


def on_gpu(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def batch(n, longest, bs, seed, grow=3, shrink=0.2, width=None, spare=50):
    """Random requests whose blocks are a permutation, and the free rest as a stack."""
    r = random.Random(seed)
    cached = [r.choice((0, 1, bs - 1, bs, bs + 1, longest, r.randint(0, longest))) for _ in range(n)]
    cached = [min(c, longest) for c in cached]
    wanted = [r.randint(0, c) if r.random() < shrink else c + r.randint(0, grow) for c in cached]
    width = width or -(-(longest + grow) // bs)
    blocks = list(range(sum(-(-c // bs) for c in cached) + spare))
    r.shuffle(blocks)
    tables = [[blocks.pop() for _ in range(-(-c // bs))] for c in cached]
    tables = [t + [-1] * (width - len(t)) for t in tables]
    return tables, cached, wanted, blocks


def check(ops, tables, cached, wanted, stack, bs, max_tokens, num_slots=None, capacity=None, num_free=None, mask=None, what=""):
    capacity = len(stack) + 100 if capacity is None else capacity
    num_free = len(stack) if num_free is None else num_free
    free = (stack + [-7] * capacity)[:capacity]
    num_slots = num_slots or (1 << 30)
    want = ref.batch_inputs(tables, cached, wanted, free, num_free, bs, num_slots, max_tokens, mask)
    t, f = on_gpu(tables) if tables else torch.zeros(0, 4, dtype=torch.int32, device=DEV), on_gpu(free)
    args = (t, on_gpu(cached), on_gpu(wanted), f, on_gpu([num_free]), bs, num_slots, max_tokens)
    for again in range(2):  # the same call on the same state gives the same
        got = ops.batch_inputs(*args, tree_mask=None if mask is None else mask.to(DEV))
        assert t.tolist() == want[0], f"{what} tables {again}"
        assert f.tolist() == want[1], f"{what} stack {again}"
        for name, g, w in zip(got._fields, got, want[2:]):
            assert g.tolist() == w, f"{what} {name} {again}"
    return got, want


@pytest.mark.parametrize("n", [0, 1, 2, 31, 33, 512, 513, 1500, 8192])
@pytest.mark.parametrize("bs", [1, 16, 48, 256])
def test_batches_of_all_sizes(ops, n, bs):
    tables, cached, wanted, stack = batch(n, 300 if n < 2000 else 60, bs, seed=n * 7 + bs, spare=4 * n + 1)
    check(ops, tables, cached, wanted, stack, bs, sum(max(0, w - c) for c, w in zip(cached, wanted)) + 5)


@pytest.mark.parametrize("spare", [0, 1, 2, 3, 5, 8, 40])
def test_too_few_blocks(ops, spare):
    """Requests are served in order while there are blocks, those that need none always; the others keep their place without slots."""
    tables, cached, wanted, stack = batch(40, 100, 16, seed=spare, grow=40, shrink=0.1, spare=spare)
    got, want = check(ops, tables, cached, wanted, stack, 16, 3000)
    held = [i for i, (c, w, n) in enumerate(zip(cached, wanted, want[7])) if n != w]
    assert held or spare >= 40


@pytest.mark.parametrize("room", [0, 1, 17, 100, 400])
def test_too_little_room_for_tokens(ops, room):
    tables, cached, wanted, stack = batch(30, 200, 16, seed=room, grow=30, spare=200)
    check(ops, tables, cached, wanted, stack, 16, room)


def test_all_requests_finish(ops):
    tables, cached, wanted, stack = batch(64, 500, 16, seed=3, spare=7)
    got, _ = check(ops, tables, cached, [0] * 64, stack, 16, 10, capacity=len(stack) + sum(-(-c // 16) for c in cached))
    assert got.num_free.item() == len(stack) + sum(-(-c // 16) for c in cached)


def test_one_request_takes_what_another_gives(ops):
    got, _ = check(ops, [[4, 5, 6, -1], [1, -1, -1, -1]], [40, 10], [0, 60], [], 16, 64)
    assert got.num_free.item() == 0 and got.slot_mapping[6:22].tolist() == [6 * 16 + i for i in range(16)]


def test_a_stack_without_room_for_what_comes_back(ops):
    check(ops, [[4, 5, 6], [1, 2, 3]], [48, 48], [0, 0], [9], 16, 8, capacity=3)


@pytest.mark.parametrize("cached, wanted", [([-1, 5], [3, 6]), ([5, 5], [-2, 6]), ([5, 70], [6, 71]), ([5, 64], [6, 65]), ([2 ** 31 - 1, 5], [-2 ** 31, 6]), ([64, 64], [64, 0])])
def test_lengths_that_no_table_holds(ops, cached, wanted):
    check(ops, [[0, 1, 2, 3], [4, 5, 6, 7]], cached, wanted, [8, 9], 16, 8)


@pytest.mark.parametrize("num_free", [-5, 0, 2, 3, 9])
def test_a_height_outside_the_stack(ops, num_free):
    check(ops, [[0, -1], [1, -1]], [16, 16], [17, 17], [8, 9, 7], 16, 8, capacity=3, num_free=num_free)


def test_bad_blocks_get_no_slot(ops):
    check(ops, [[-1, -1], [1, -1], [99, -1], [3, -1]], [1, 15, 1, 16], [2, 17, 2, 17], [-3, 50], 16, 8, num_slots=160)


@pytest.mark.parametrize("words", [1, 2])
def test_positions_of_trees_follow_the_depth(ops, words):
    r = random.Random(words)
    counts = [r.randint(0, 64 * words) for _ in range(11)]
    mask = ref.trees(counts, words, seed=words)
    mask[3] = 0  # a node that sees nothing stays at the tree's beginning
    mask[4:9] = -1  # bits past the tree are ignored: no position lies behind the tree's last place
    cached = [r.randint(0, 90) for _ in counts]
    wanted = [c + t for c, t in zip(cached, counts)]
    got, _ = check(ops, [[i * 16 + j for j in range(16)] for i in range(11)], cached, wanted, list(range(200, 300)), 16, sum(counts), mask=mask)
    first = torch.tensor(cached).repeat_interleave(torch.tensor(counts))
    last = torch.tensor(wanted).repeat_interleave(torch.tensor(counts)) - 1
    assert ((got.positions.cpu() >= first) & (got.positions.cpu() <= last)).all()


@pytest.mark.parametrize("bs, width", [(2 ** 31 - 1, 1), (2 ** 30, 1), (715827882, 3), (16, (2 ** 31 - 1) // 16)])
def test_the_longest_rows(ops, bs, width):
    full = bs * width
    tables = torch.zeros(1, width, dtype=torch.int32, device=DEV)
    got = ops.batch_inputs(tables, on_gpu([full - 9]), on_gpu([full]), on_gpu([5]), on_gpu([1]), bs, 2 ** 31 - 1, 12)
    assert got.positions.tolist() == list(range(full - 9, full)) + [0] * 3 and got.context_lens.tolist() == [full] and got.num_free.tolist() == [1]
    place = (full - 9) % bs
    assert got.slot_mapping.tolist() == list(range(place, place + 9)) + [-1] * 3


def test_rows_of_a_wider_table_and_a_wider_mask(ops):
    big = torch.full((5, 40), -9, dtype=torch.int32, device=DEV)
    tables = big[:, 3:9]
    tables.copy_(on_gpu([[10 * i + j for j in range(6)] for i in range(5)]))
    mask = torch.full((50, 4), 7, dtype=torch.int64, device=DEV)[:, 1:2]
    got = ops.batch_inputs(tables, on_gpu([3] * 5), on_gpu([3, 4, 20, 0, 40]), on_gpu([90, 91, 92, 93]), on_gpu([4]), 16, 4000, 50, tree_mask=mask)
    # rows of 0, 1, 17, 0 and 37 new tokens: the last does not fit behind the others
    assert got.cu_seqlens_q.tolist() == [0, 0, 1, 18, 18, 18] and got.context_lens.tolist() == [3, 4, 20, 0, 3]
    # row 3 gives its block 30 back; row 2 takes it
    assert got.slot_mapping.tolist() == [10 * 16 + 3] + [20 * 16 + i for i in range(3, 16)] + [30 * 16 + i for i in range(4)] + [-1] * 32
    assert got.num_free.tolist() == [4]
    untouched = torch.cat([big[:, :3], big[:, 9:]], 1)
    assert (untouched == -9).all()
    assert got.positions.tolist() == [3] + [5] * 17 + [0] * 32  # one node sees itself only, the others three


def test_a_captured_call_serves_later_batches(ops):
    tables, cached, wanted, stack = batch(37, 300, 16, seed=5, spare=100)
    t, c, w, f, n = on_gpu(tables), on_gpu(cached), on_gpu(wanted), on_gpu(stack + [-1] * 200), on_gpu([len(stack)])
    ops.batch_inputs(t, c, w, f, n, 16, 1 << 20, 128)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.batch_inputs(t, c, w, f, n, 16, 1 << 20, 128)
        c.copy_(got.context_lens)  # the next step's state
        n.copy_(got.num_free)
    t.copy_(on_gpu(tables))
    c.copy_(on_gpu(cached))
    n.copy_(on_gpu([len(stack)]))
    f.copy_(on_gpu(stack + [-1] * 200))
    state = (tables, cached, stack + [-1] * 200, len(stack))
    r = random.Random(8)
    for step in range(12):
        wanted = [0 if r.random() < 0.1 else min(x + r.randint(0, 3), 300) for x in state[1]]
        w.copy_(on_gpu(wanted))
        graph.replay()
        want = ref.batch_inputs(state[0], state[1], wanted, state[2], state[3], 16, 1 << 20, 128)
        assert t.tolist() == want[0], f"step {step}"
        for name, g, e in zip(got._fields, got, want[2:]):
            assert g.tolist() == e, f"step {step} {name}"
        assert c.tolist() == want[7] and f[:want[8][0]].tolist() == want[1][:want[8][0]]
        state = (want[0], want[7], want[1], want[8][0])


def test_on_another_stream(ops):
    tables, cached, wanted, stack = batch(64, 200, 16, seed=9, spare=99)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        check(ops, tables, cached, wanted, stack, 16, 300)
