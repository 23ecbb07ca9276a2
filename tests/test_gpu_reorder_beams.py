"""ops.reorder_beams on a B200 against its definition on the host: everything it moves is compared bit by bit."""
import random

import pytest
import torch

import beam_util as ref
import gpu_util

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def ops(pkg):
    gpu_util.ensure_group()
    torch.cuda.set_device(0)
    pkg.init_runtime(max_tokens=512, hidden=1024, vocab=2048, max_seqs=64)
    from nanovllm_b200 import ops
    yield ops
    pkg.shutdown_runtime()


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


class Case:
    """Requests of `beams` rows that came apart from one another: row b has the blocks of an earlier row up to a random place."""

    def __init__(self, requests, beams, longest, bs, width=None, shared=0, seed=0, spare=None, layers=2, shape=(2, 64), dtype=torch.bfloat16, dead=0.15, history=None):
        r = random.Random(seed)
        self.bs, self.n, self.beams = bs, requests, beams
        self.width = width if width is not None else -(-longest // bs) + 1
        number, self.tables, self.lens, self.first = shared, [], [], []
        for _ in range(requests):
            mine, longs = [], []
            first = r.randint(0, shared)
            for b in range(beams):
                n = r.choice((0, r.randint(0, longest), longest, max(0, longest - bs), longest // bs * bs))
                table = list(range(first))[:n // bs]
                if b > 0 and r.random() < 0.8:
                    a = r.randrange(b)
                    common = r.randint(0, min(n, longs[a])) // bs
                    table = mine[a][:common] if common > len(table) else table
                    # now and then the same open block as well (both were just made from one row)
                    if common == longs[a] // bs and n // bs == common and n % bs and longs[a] % bs and r.random() < 0.5:
                        table = mine[a][:common + 1]
                        n = longs[a]
                fresh = -(-n // bs) - len(table)
                table = table + list(range(number, number + fresh))
                number += fresh
                mine.append(table)
                longs.append(n)
            for table in mine:
                self.tables.append(table + [r.choice((-1, 2 ** 31 - 1, -7, 0)) for _ in range(self.width - len(table))])
            self.lens += longs
            self.first.append(first)
        spare = spare if spare is not None else requests * beams
        self.blocks = number + spare + 2
        order = list(range(self.blocks))
        r.shuffle(order)
        self.tables = [[order[b] if 0 <= b < number and c < -(-n // bs) else b for c, b in enumerate(row)] for row, n in zip(self.tables, self.lens)]
        self.num_free = spare
        self.free = [order[b] for b in range(number, number + spare)] + [-1] * (number + 2)
        self.parents = [[-1 if r.random() < dead else r.randrange(beams) for _ in range(beams)] for _ in range(requests)]
        g = torch.Generator().manual_seed(seed)
        raw = torch.randint(-128, 128, (2, layers, self.blocks, bs, *shape, torch.empty(0, dtype=dtype).element_size()), generator=g, dtype=torch.int8)
        self.cache = raw.to(DEV).view(dtype).squeeze(-1)
        self.history = self.said = self.tokens = None
        if history is not None:
            rows = requests * beams
            self.history = torch.randint(0, 1 << 40, (rows, history), generator=g).to(DEV)
            self.said = [r.choice((0, history, max(0, history - 1), r.randint(0, history))) for _ in range(rows)]
            self.tokens = [[r.choice((-1, r.randint(0, 1 << 40), 7)) for _ in range(beams)] for _ in range(requests)]

    def run(self, ops, **change):
        a = dict(parents=i32(self.parents).view(self.n, self.beams), block_tables=i32(self.tables).view(self.n * self.beams, self.width), context_lens=i32(self.lens), free_blocks=i32(self.free),
                 num_free=i32([self.num_free]), kv_cache=self.cache.clone(), first_blocks=i32(self.first))
        if self.history is not None:
            a.update(history=self.history, history_lens=i32(self.said), tokens=None if self.tokens is None else torch.tensor(self.tokens, device=DEV).view(self.n, self.beams))
        a.update(change)
        return a, ops.reorder_beams(**a)

    def check(self, a, out):
        tables, lens, stack, height, copies = ref.reorder_beams(self.parents, self.tables, self.lens, self.free, self.num_free, self.bs, self.blocks, self.first)
        assert out.block_tables.tolist() == tables
        assert out.context_lens.tolist() == lens
        assert out.num_free.tolist() == [height]
        assert a["free_blocks"].tolist()[:height] == stack[:height]
        want = self.cache.clone()
        for source, to, tokens in copies:
            want[:, :, to, :tokens] = self.cache[:, :, source, :tokens]
        assert torch.equal(a["kv_cache"].view(torch.int8), want.view(torch.int8))
        if self.history is None:
            assert out.history is None and out.history_lens is None
        else:
            text, said = ref.append_history(self.parents, self.history.tolist(), self.said, self.tokens, self.history.shape[1])
            assert out.history.tolist() == text and out.history_lens.tolist() == said
        return copies


@pytest.mark.parametrize("requests, beams, longest, bs", [(1, 1, 1, 1), (1, 1, 0, 16), (1, 4, 40, 16), (2, 5, 3, 7), (3, 32, 50, 16), (5, 2, 200, 1), (7, 29, 133, 48), (40, 8, 70, 16), (2, 16, 999, 3),
                                                         (2, 9, 4000, 16), (4, 8, 1030, 4), (3, 17, 129, 2), (130, 3, 33, 16), (1, 3, 5000, 5)])
@pytest.mark.parametrize("shared", [0, 3])
def test_sizes(ops, requests, beams, longest, bs, shared):
    for seed in range(3):
        case = Case(requests, beams, longest, bs, shared=shared, seed=seed, width=max(shared, -(-longest // bs)) + 1, shape=(1, 8), history=13)
        case.check(*case.run(ops))


@pytest.mark.parametrize("bs, shape, dtype", [(16, (8, 128), torch.bfloat16), (256, (2, 64), torch.bfloat16), (48, (3, 128), torch.bfloat16), (16, (1, 16), torch.uint8), (5, (1, 4), torch.float32),
                                             (64, (3, 8), torch.float16)])
def test_caches(ops, bs, shape, dtype):
    case = Case(6, 5, 3 * bs + 1, bs, seed=bs, layers=3, shape=shape, dtype=dtype)
    a, out = case.run(ops)
    assert case.check(a, out), "nothing was copied"


@pytest.mark.parametrize("spare", [0, 1, 3])
def test_not_enough_blocks(ops, spare):
    """Copies beyond the stack's blocks are not made: the rows lose the tokens of their last block."""
    for seed in range(6):
        case = Case(4, 6, 40, 16, seed=seed, spare=spare, dead=0.0)
        case.parents = [[random.Random(seed).randrange(2)] * 6 if r % 2 else p for r, p in enumerate(case.parents)]
        case.check(*case.run(ops))
    # (above, the blocks that are given back mostly do; here there are none of them)
    case = Case(3, 6, 40, 16, seed=9, spare=spare, dead=0.0, history=4)
    case.parents = [[0] * 6 for _ in range(3)]
    case.lens = [33 if i % 6 == 0 else 0 for i in range(18)]
    for r in range(3):
        case.tables[6 * r][:3] = [3 * r, 3 * r + 1, 3 * r + 2]
    case.free = [b for b in range(9, 9 + spare)] + [-1] * 4
    a, out = case.run(ops)
    assert len(case.check(a, out)) == spare
    assert out.context_lens.tolist().count(32) == 15 - spare


def test_all_from_one_and_each_its_own(ops):
    for parents in ([0, 0, 0, 0], [3, 3, 3, 3], [0, 1, 2, 3], [3, 2, 1, 0], [-1, -1, -1, -1], [4, -5, 2 ** 31 - 1, 1]):
        case = Case(3, 4, 100, 16, seed=1, shared=2, history=5)
        case.parents = [list(parents)] * 3
        case.check(*case.run(ops))


def test_a_stack_that_is_full_or_holds_anything(ops):
    """Heights outside the stack, block numbers outside the cache, on the stack and in the tables."""
    case = Case(3, 4, 100, 16, seed=2)
    for num_free in (-4, 0, 2, 10 ** 9):
        case.num_free = num_free
        case.check(*case.run(ops))
    case = Case(3, 4, 100, 16, seed=3)
    case.free = [-1, case.blocks, 2 ** 31 - 1, -2 ** 31] * 4
    case.num_free = 7
    case.check(*case.run(ops))
    case = Case(3, 4, 100, 16, seed=4, shared=1)
    case.tables[2][1] = case.tables[5][0] = -1
    case.tables[7][3] = case.blocks
    case.tables[9][2] = 2 ** 31 - 1
    case.first = [-3, 10 ** 9, 1]
    case.check(*case.run(ops))
    case.lens[1], case.lens[6], case.lens[11] = -1, 10 ** 9, 2 ** 31 - 1
    case.check(*case.run(ops))
    empty = Case(2, 3, 30, 16, seed=5)
    empty.free, empty.num_free = [], 0
    empty.check(*empty.run(ops, free_blocks=torch.zeros(0, dtype=torch.int32, device=DEV)))


def test_layouts(ops):
    """Tables and histories inside wider tensors; one layer of a cache; a cache whose layers are further apart than they are large; no cache at all."""
    case = Case(3, 5, 80, 16, seed=6, history=9)
    rows = 15
    tables = torch.full((rows, case.width + 5), -9, dtype=torch.int32, device=DEV)
    tables[:, 2:-3] = i32(case.tables)
    history = torch.full((rows, 13), -9, dtype=torch.int64, device=DEV)
    history[:, 1:10] = case.history
    case.check(*case.run(ops, block_tables=tables[:, 2:-3], history=history[:, 1:10]))
    wide = torch.zeros(2, 2, case.blocks + 3, *case.cache.shape[3:], dtype=torch.bfloat16, device=DEV)
    inside = wide[:, :, :case.blocks]
    inside.copy_(case.cache)
    case.check(*case.run(ops, kv_cache=inside))
    assert not wide[:, :, case.blocks:].any()
    one = case.cache[1, 0].clone()
    _, want = case.run(ops)
    a, out = case.run(ops, kv_cache=one)
    assert torch.equal(out.block_tables, want.block_tables)
    case.cache = case.cache[1:, :1]
    case.check(dict(a, kv_cache=one[None, None]), out)
    none = torch.zeros(0, *case.cache.shape[2:], dtype=torch.bfloat16, device=DEV)
    assert torch.equal(case.run(ops, kv_cache=none)[1].block_tables, want.block_tables)


def test_histories(ops):
    """Lengths that the width does not hold, no tokens, histories of no width, long ones."""
    for width in (0, 1, 1023, 1024, 1025, 5000):
        case = Case(3, 3, 20, 16, seed=width, history=width)
        case.said[0], case.said[1] = -4, 10 ** 6
        case.check(*case.run(ops))
        case.tokens = None
        case.check(*case.run(ops))


def test_no_requests(ops):
    out = ops.reorder_beams(torch.zeros(0, 4, dtype=torch.int32, device=DEV), torch.zeros(0, 3, dtype=torch.int32, device=DEV), i32([]), i32([4, 5, 6]), i32([2]),
                            torch.zeros(2, 16, 1, 8, dtype=torch.bfloat16, device=DEV))
    assert out.num_free.tolist() == [2] and out.block_tables.shape == (0, 3)


def test_many_copies(ops):
    """More copies than a CTA lists at a time."""
    case = Case(60, 32, 33, 16, seed=7, shape=(1, 8), dead=0.0)
    case.parents = [[0] * 32 for _ in range(60)]
    case.lens = [n if i % 32 else 33 for i, n in enumerate(case.lens)]
    number = case.blocks
    for i in range(0, len(case.tables), 32):
        case.tables[i] = [number, number + 1, number + 2] + case.tables[i][3:]
        number += 3
    case.blocks = number
    case.cache = torch.randint(-9, 9, (2, 2, number, 16, 1, 8), device=DEV).bfloat16()
    a, out = case.run(ops)
    assert len(case.check(a, out)) == 60 * 31


def test_captured_and_on_two_streams(ops):
    """Two graphs on two streams at the same time, each with its stack and cache; the same call again gives the same results."""
    cases = [Case(5, 6, 90, 16, seed=8, history=30), Case(3, 9, 300, 48, seed=9, shared=2, history=8)]
    streams, graphs, work = [torch.cuda.Stream() for _ in cases], [], []
    for case, s in zip(cases, streams):
        a, _ = case.run(ops)
        torch.cuda.synchronize()
        a["free_blocks"].copy_(i32(case.free))
        a["kv_cache"].copy_(case.cache)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = ops.reorder_beams(**a)
        graphs.append(graph)
        work.append((a, out))
    for _ in range(2):
        for (a, _), case in zip(work, cases):
            r = random.Random(len(work))
            a["parents"].copy_(i32(case.parents))
        torch.cuda.synchronize()
        for _ in range(2):  # (a replay finds the stack's places below num_free, and the blocks that are copied from, as they were)
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for case, (a, out) in zip(cases, work):
            case.check(a, out)
            a["kv_cache"].copy_(case.cache)
            a["free_blocks"].copy_(i32(case.free))
            case.parents = [p[1:] + p[:1] for p in case.parents]
