"""ops.reorder_beams on a B200: tokens of any negative value, and rows of which one goes on in a block that is full in another."""
import random

import pytest
import torch

import gpu_util
from tests.test_gpu_reorder_beams import Case, i32

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


@pytest.mark.parametrize("width", [1, 9, 1025])
def test_a_negative_token_is_none_whatever_its_value(ops, width):
    """Behind a row's tokens there is -1, whatever negative number stood for "none"."""
    case = Case(4, 5, 40, 16, seed=width, history=width)
    r = random.Random(width)
    case.tokens = [[r.choice((-2, -100, -2 ** 31, -2 ** 40, -2 ** 63, 0, 2 ** 62)) for _ in range(5)] for _ in range(4)]
    assert min(min(t) for t in case.tokens) < -1
    case.check(*case.run(ops))


class Prefixes:
    """Rows of a request that are beginnings of one another: a tree of blocks, in which a row may end anywhere."""

    def __init__(self, requests, beams, bs, seed):
        r = random.Random(seed)
        self.bs, self.beams, number = bs, beams, 0
        self.tables, self.lens = [], []
        for _ in range(requests):
            mine, longs = [], []
            for b in range(beams):
                if b > 0 and r.random() < 0.8:
                    a = r.randrange(b)
                    n, table = r.randint(0, longs[a]), list(mine[a])  # a beginning of row a
                    table = table[:-(-n // bs)]
                    if r.random() < 0.5 and n % bs == 0:  # ... that goes on by itself
                        more = r.randint(0, 2 * bs)
                        table += range(number, number + -(-more // bs))
                        number += -(-more // bs)
                        n += more
                else:
                    n = r.randint(0, 5 * bs)
                    table = list(range(number, number + -(-n // bs)))
                    number += len(table)
                mine.append(table)
                longs.append(n)
            order = list(range(beams))
            r.shuffle(order)  # (a row with more tokens comes before one with fewer as often as behind it)
            self.tables += [mine[i] for i in order]
            self.lens += [longs[i] for i in order]
        self.width = max(len(t) for t in self.tables) + 1
        self.blocks = number + requests * beams
        order = list(range(self.blocks))
        r.shuffle(order)
        self.tables = [[order[x] for x in t] for t in self.tables]
        self.free = [order[x] for x in range(number, self.blocks)]
        self.parents = [[b if r.random() < 0.6 else r.randrange(-1, beams) for b in range(beams)] for _ in range(requests)]


@pytest.mark.parametrize("requests, beams, bs", [(1, 3, 16), (5, 4, 16), (9, 8, 3), (3, 17, 5), (2, 32, 16)])
def test_an_open_block_is_no_other_rows(ops, requests, beams, bs):
    """What a row goes on in is its own: where another row has it, open as well or full, one of them has a copy.  Each row reads what its parent read, and no block is lost."""
    shared = 0
    for seed in range(8):
        case = Prefixes(requests, beams, bs, seed)
        rows = requests * beams
        tables = torch.full((rows, case.width), -1, dtype=torch.int32)
        for row, t in enumerate(case.tables):
            tables[row, :len(t)] = torch.tensor(t, dtype=torch.int32)
        cache = torch.randint(-2 ** 31, 2 ** 31 - 1, (2, case.blocks, bs, 1, 4), generator=torch.Generator().manual_seed(seed), dtype=torch.int32)
        stack = torch.tensor(case.free + [-1] * (case.blocks - len(case.free)), dtype=torch.int32, device=DEV)
        after = cache.to(DEV)
        out = ops.reorder_beams(i32(case.parents), tables.to(DEV), i32(case.lens), stack, i32([len(case.free)]), after)
        after, new, lens, height = after.cpu(), out.block_tables.tolist(), out.context_lens.tolist(), out.num_free.item()
        used = []  # per request: (column, block), and the rows that have it, each with whether it goes on in it
        for r in range(requests):
            held = {}
            for b in range(beams):
                row, p = r * beams + b, case.parents[r][b]
                n = case.lens[r * beams + p] if p >= 0 else 0
                assert lens[row] == n
                have = -(-n // bs)
                assert min(new[row][:have], default=0) >= 0 and new[row][have:] == [-1] * (case.width - have)
                for i in range(n):
                    assert torch.equal(after[:, new[row][i // bs], i % bs], cache[:, case.tables[r * beams + p][i // bs], i % bs])
                for c in range(have):
                    held.setdefault((c, new[row][c]), []).append(c == n // bs)
                    shared += c < n // bs and any(c == case.lens[r * beams + q] // bs and case.tables[r * beams + q][c:c + 1] == case.tables[r * beams + p][c:c + 1] for q in case.parents[r] if q >= 0)
            assert all(len(x) == 1 for x in held.values() if any(x)), "a block that one row goes on in is another's as well"
            used += [block for _, block in held]
        left = stack.tolist()[:height]
        # (blocks of rows that nobody continues come back; the tree's blocks were each some row's)
        assert len(set(used)) == len(used) and len(set(left)) == height and not set(left) & set(used)
        assert set(left) | set(used) == {x for t in case.tables for x in t} | set(case.free)
    assert shared or requests * beams < 10, "no row's open block was full in another"
