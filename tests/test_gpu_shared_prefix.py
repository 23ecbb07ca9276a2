"""ops.shared_prefix_attention on a B200 against its definition in 64 bits on the same bf16 inputs.

Tolerance, per element.  Rounding: the probabilities are rounded to bf16 for the second product, each by at most 2^-8 of itself, while their
sum is taken before: sum p (1 + e) v / sum p is off by at most 2^-8 A with A = sum p |v| / sum p, and the result's own rounding adds
2^-8 (|o| + that).  What is done in 32 bits: a score is a sum of head_dim <= 128 products, off by at most 128 * 2^-24 = 2^-17 of
S = |scale| * sum |q k|, which is about 11 for the draws here (standard deviations of 1.5 and 1), so by 2^-13, and p by that part of itself in the numerator and in
the sum below; exp2's argument and result add 2^-21 and less; sums over n keys add at most 2^-24 of A for every step of 64 keys (2^-15 at 32768).
Together below 2^-11 A, and 2^-10 A leaves room for scores of twice that size."""
import random

import pytest
import torch

import beam_util as ref
import gpu_util

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = torch.finfo(torch.bfloat16).eps / 2  # 2^-8
FP32 = 2.0 ** -10


@pytest.fixture(scope="module")
def rt(pkg):
    gpu_util.ensure_group()
    torch.cuda.set_device(0)
    runtime = pkg.init_runtime(max_tokens=512, hidden=1024, vocab=2048, max_seqs=64)
    yield runtime
    pkg.shutdown_runtime()


@pytest.fixture(scope="module")
def ops(pkg, rt):
    from nanovllm_b200 import ops
    return ops


@pytest.fixture(autouse=True)
def no_wait_has_run_out(rt):
    yield
    torch.cuda.synchronize()
    rt.check_status()


class Case:
    """groups: (tokens in common, [each sequence's tokens in all]); 0 tokens: a padded row, whose table is garbage.  Other places of the cache hold NaN."""

    def __init__(self, groups, nq=4, nkv=2, hd=128, bs=16, seed=0, before=0, behind=0, std=1.5, scale=None):
        g = torch.Generator(device=DEV).manual_seed(seed)
        r = random.Random(seed)
        self.bs, self.scale = bs, hd ** -0.5 if scale is None else scale
        self.lens, self.cu, self.prefix, chains = [5] * before, [before], [], [(None, 5)] * before
        for common, lens in groups:
            self.lens += lens
            self.cu.append(len(self.lens))
            full = min([common] + [n for n in lens if n > 0]) // bs * bs
            self.prefix.append(full)
            chains += [(len(self.prefix), n) for n in lens]
        self.lens += [7] * behind
        chains += [(None, 7)] * behind
        n, width = len(self.lens), max(1, max(-(-l // bs) for l in self.lens)) + 1
        used = sum(-(-l // bs) for l in self.lens) + 5
        order = list(range(used))
        r.shuffle(order)
        shared, self.tables = {}, []
        for s, (group, length) in enumerate(chains):
            mine = []
            if group is not None and length > 0:
                whole = self.prefix[group - 1] // bs
                if group not in shared:
                    shared[group] = [order.pop() for _ in range(whole)]
                mine = list(shared[group])
            mine += [order.pop() for _ in range(-(-length // bs) - len(mine))]
            self.tables.append(mine + [r.choice((-1, 2 ** 31 - 1, -2 ** 31, 10 ** 6)) for _ in range(width - len(mine))])
        self.k = torch.full((used, bs, nkv, hd), float("nan"), dtype=torch.bfloat16, device=DEV)
        self.v = torch.full((used, bs, nkv, hd), float("nan"), dtype=torch.bfloat16, device=DEV)
        for s, length in enumerate(self.lens):
            for c in range(-(-length // bs)):
                t = min(bs, length - c * bs)
                for x in (self.k, self.v):
                    x[self.tables[s][c], :t] = torch.empty(t, nkv, hd, device=DEV).normal_(generator=g).bfloat16()
        self.q = torch.empty(n, nq, hd, device=DEV).normal_(0, std, generator=g).bfloat16()
        self.largest = max(b - a for a, b in zip(self.cu, self.cu[1:])) if groups else 0

    def args(self, **change):
        i = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
        a = dict(q=self.q, k_cache=self.k, v_cache=self.v, cu_groups=i(self.cu), prefix_lens=i(self.prefix), context_lens=i(self.lens), block_tables=i(self.tables),
                 max_group=self.largest, scale=self.scale)
        a.update(change)
        return a

    def expected(self):
        return ref.shared_prefix_attention(self.q, self.k, self.v, self.cu, self.lens, self.tables, self.scale)

    def check(self, got):
        want, size = self.expected()
        assert got.shape == self.q.shape and got.dtype == torch.bfloat16
        bound = HALF * size + HALF * (want.abs() + HALF * size) + FP32 * size
        err = (got.double() - want).abs()
        assert torch.isfinite(got).all()
        worst = ((err - bound) / (bound + 1e-30)).flatten(1).max(1).values
        assert (err <= bound).all(), f"sequences {(worst > 0).nonzero().flatten().tolist()}, {worst.max().item() + 1:.2f} times the bound"


SHAPES = [(4, 2, 128, 16), (8, 8, 64, 48), (5, 1, 128, 32), (16, 2, 64, 16), (9, 1, 64, 64), (48, 4, 128, 16), (32, 1, 128, 16), (40, 2, 64, 256), (128, 1, 64, 16), (33, 1, 128, 112)]


@pytest.mark.parametrize("nq, nkv, hd, bs", SHAPES)
def test_shapes(ops, nq, nkv, hd, bs):
    """One to 128 heads per KV head, in blocks that divide a tile or do not; groups with and without common tiles, of one sequence, of none, rows of no group."""
    case = Case([(300, [300, 301, 431, 700]), (70, [71]), (200, [200, 333, 0, 201]), (0, [1, 64, 65]), (63, [90, 63]), (128, []), (640, [650] * 5)], nq, nkv, hd, bs, seed=nq + hd, before=2, behind=3)
    case.check(ops.shared_prefix_attention(**case.args()))


@pytest.mark.parametrize("lens", [[1], [1, 1], [0], [0, 0, 0], [64], [63, 64, 65], [16, 0, 17], [0, 128, 129], [128, 0, 128], [1, 4000], [4000, 4000], [191, 192, 193]])
@pytest.mark.parametrize("nq", [2, 24])
def test_lengths(ops, lens, nq):
    """One group whose common tokens are all that its shortest sequence has: nothing, one token, tiles to the last token."""
    live = [n for n in lens if n > 0]
    case = Case([(min(live, default=0), lens)], nq, 2, 128, 16, seed=sum(lens) + nq)
    got = ops.shared_prefix_attention(**case.args())
    case.check(got)
    assert all(not got[i].any() for i, n in enumerate(lens) if n == 0)


@pytest.mark.parametrize("lens", [[1], [100, 512, 3], [0, 7], [257] * 9])
@pytest.mark.parametrize("nq, hd", [(2, 128), (32, 64)])
def test_short_tables(ops, lens, nq, hd):
    """Tables of at most eight tiles with few sequences: every sequence is walked by one CTA."""
    case = Case([(max(lens) if len(set(lens)) == 1 else 0, lens)], nq, 2, hd, 256, seed=len(lens) + hd)
    case.tables = [row[:2] for row in case.tables]
    case.check(ops.shared_prefix_attention(**case.args()))


@pytest.mark.parametrize("size, nq, hd", [(300, 8, 64), (128, 2, 128), (129, 1, 64), (17, 16, 128)])
def test_many_sequences(ops, size, nq, hd):
    """More sequences than the tensor core's rows hold: several items per group, the last of them not full."""
    r = random.Random(size)
    case = Case([(512, [512 + r.randint(0, 150) for _ in range(size)])], nq, 1, hd, 64, seed=size)
    case.check(ops.shared_prefix_attention(**case.args()))


@pytest.mark.parametrize("scale", [0.0, -0.09, 1.0])
def test_scales(ops, scale):
    """Of either sign, zero (every key counts the same), and large: S is 1.0 * 128 products of |q k| of 1.5 (2/pi) on average, about 122 and in ten standard deviations
    of the sum (1.2 each) 140, times 2^-17 = 2^-9.9: FP32 of A and as much in the sum, which the bound's 2^-7 covers where p is not that of one key alone."""
    case = Case([(200, [210, 300, 520])], 6, 2, 128, 16, seed=4, scale=scale, std=1.0 if scale == 1.0 else 1.5)
    case.check(ops.shared_prefix_attention(**case.args()))


def test_scores_that_grow_and_fall(ops):
    """Keys whose scores rise by hundreds from tile to tile, and others that fall: the running maximum moves in every tile, in both kinds of keys."""
    for order in (1, -1):
        case = Case([(640, [640, 700, 1500])], 4, 2, 128, 16, seed=5)
        unit = torch.ones(128, device=DEV, dtype=torch.bfloat16)
        case.q[:] = unit
        for s, length in enumerate(case.lens):
            for i in range(length):
                # (a key's score: 128 times its one value times 2^-7 = 1.0 for value 1: exact in bf16 and in 32 bits)
                case.k[case.tables[s][i // 16], i % 16] = float(order * (i // 64) * 16)
        case.scale = 2.0 ** -7
        case.check(ops.shared_prefix_attention(**case.args()))


def test_keys_that_do_not_count_may_be_anything(ops):
    """Infinities and NaN behind the contexts change no bit of the result; nor does what a padded row's table says."""
    case = Case([(130, [131, 150, 0, 299]), (16, [17, 40])], 10, 2, 64, 16, seed=6)
    got = ops.shared_prefix_attention(**case.args())
    case.check(got)
    for value in (float("inf"), -float("inf"), 3e38, 0.0):
        for x in (case.k, case.v):
            x[x.isnan() | x.isinf() | (x == 0) | (x.abs() > 1e38)] = value
        case.tables[2] = [random.Random(1).randrange(5)] * len(case.tables[2])
        assert torch.equal(ops.shared_prefix_attention(**case.args()), got)


def test_layouts_and_orders(ops):
    """Queries inside a wider tensor, tables inside a wider one, groups that do not begin at sequence 0."""
    case = Case([(160, [170, 190]), (96, [100, 300, 97])], 8, 4, 128, 32, seed=7, before=1, behind=2)
    want = ops.shared_prefix_attention(**case.args())
    case.check(want)
    n, nq, hd = case.q.shape
    wide = torch.full((n, 3 * nq * hd + 8), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide[:, 8:8 + nq * hd] = case.q.view(n, -1)
    q = wide[:, 8:8 + nq * hd].view(n, nq, hd)
    tables = torch.full((n, len(case.tables[0]) + 3), -1, dtype=torch.int32, device=DEV)
    tables[:, 1:-2] = torch.tensor(case.tables, dtype=torch.int32, device=DEV)
    assert torch.equal(ops.shared_prefix_attention(**case.args(q=q, block_tables=tables[:, 1:-2])), want)


def test_a_prefix_that_a_shorter_context_cuts(ops):
    """prefix_lens beyond the shortest context of the group, beyond all of them, negative: the result is the contexts' own."""
    case = Case([(320, [320, 400, 700])], 4, 2, 128, 16, seed=8)
    for prefix in (10 ** 9, 320, 319, 64, 63, 0, -5):
        if prefix > 320:
            case.lens = [320, 200, 150]  # tables agree in 320 tokens
        case.check(ops.shared_prefix_attention(**case.args(prefix_lens=torch.tensor([prefix], dtype=torch.int32, device=DEV))))
        case.lens = [320, 400, 700]


def test_lengths_that_tables_do_not_hold(ops):
    """Negative lengths count as none, longer ones end with the table; bounds of groups outside the batch are cut."""
    case = Case([(64, [64, 100, 80])], 4, 2, 128, 16, seed=9)
    case.tables = [row[:-1] if i == 1 else (row[:len(case.tables[1]) - 1]) for i, row in enumerate(case.tables)]
    full = len(case.tables[1]) * 16
    last = case.tables[1][-1]
    case.k[last], case.v[last] = torch.randn_like(case.k[last]), torch.randn_like(case.v[last])
    got = ops.shared_prefix_attention(**case.args(context_lens=torch.tensor([-3, 10 ** 9, 80], dtype=torch.int32, device=DEV), cu_groups=torch.tensor([-2, 10 ** 6], dtype=torch.int32, device=DEV)))
    case.lens = [0, full, 80]
    case.check(got)


def test_bounds_that_fall(ops):
    """Groups that would overlap are none: every sequence sees nothing, and what is behind the result stays as it was."""
    case = Case([(128, [128, 200, 140]), (64, [64, 100])], 4, 2, 128, 16, seed=16)
    for cu in ([0, 5, 0], [3, 0, 5], [5, 5, 0], [0, 5, 2]):
        assert not ops.shared_prefix_attention(**case.args(cu_groups=torch.tensor(cu, dtype=torch.int32, device=DEV))).any()
    case.check(ops.shared_prefix_attention(**case.args()))


def test_no_sequences_and_no_groups(ops):
    case = Case([(64, [64, 100])], 4, 2, 128, 16, seed=10)
    none = case.args(cu_groups=torch.zeros(1, dtype=torch.int32, device=DEV), prefix_lens=torch.zeros(0, dtype=torch.int32, device=DEV), max_group=0)
    assert not ops.shared_prefix_attention(**none).any()
    empty = case.args(q=case.q[:0], context_lens=torch.zeros(0, dtype=torch.int32, device=DEV), block_tables=torch.zeros(0, 3, dtype=torch.int32, device=DEV))
    assert ops.shared_prefix_attention(**empty).shape == (0, 4, 128)


def test_agrees_with_paged_attention(ops):
    """The same call a sequence at a time: each of the two is within its bound of the exact result, so they are within twice that of each other."""
    case = Case([(512, [600, 530, 777]), (64, [70, 90])], 8, 4, 128, 256, seed=11)  # (blocks that both serve)
    a = case.args()
    got, plain = ops.shared_prefix_attention(**a), ops.paged_attention(case.q, case.k, case.v, a["context_lens"], a["block_tables"], case.scale)
    want, size = case.expected()
    assert ((got.double() - plain.double()).abs() <= 2 * (HALF * size + HALF * (want.abs() + HALF * size) + FP32 * size)).all()


def test_repeated_calls_agree(ops):
    case = Case([(1024, [1024 + 37 * i for i in range(12)]), (128, [200] * 9)], 16, 4, 128, 16, seed=12)
    first = ops.shared_prefix_attention(**case.args())
    for _ in range(5):
        assert torch.equal(ops.shared_prefix_attention(**case.args()), first)


def test_captured_and_on_two_streams(ops):
    """Two graphs captured on a side stream, replayed at the same time on two streams, with lengths and tables that change under them; eager calls between."""
    cases = [Case([(512, [600, 530, 777]), (64, [70, 90])], 8, 4, 128, 16, seed=13), Case([(256, [256 + 50 * i for i in range(20)])], 20, 2, 64, 16, seed=14)]
    streams, graphs, outs, args = [torch.cuda.Stream() for _ in cases], [], [], [c.args() for c in cases]
    for a, s in zip(args, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            ops.shared_prefix_attention(**a)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append(ops.shared_prefix_attention(**a))
        graphs.append(graph)
    torch.cuda.synchronize()
    for cut in (0, 33, 60, 5):
        for c, a in zip(cases, args):
            lens = [max(0, n - cut) for n in c.lens]
            a["context_lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        torch.cuda.synchronize()
        for _ in range(3):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        eager = [ops.shared_prefix_attention(**a) for a in args]
        torch.cuda.synchronize()
        for c, o, e in zip(cases, outs, eager):
            whole, c.lens = c.lens, [max(0, n - cut) for n in c.lens]
            c.check(o)
            c.lens = whole
            assert torch.equal(o, e)


def test_slots_beyond_32_bits_of_elements(ops):
    """A cache whose later blocks lie past 2^32 elements."""
    nkv, hd, bs = 8, 128, 256
    blocks = (1 << 32) // (bs * nkv * hd) + 8
    if torch.cuda.mem_get_info()[0] < 3 * blocks * bs * nkv * hd * 2:
        pytest.skip("needs 26 GB")
    case = Case([(512, [600, 530])], 16, nkv, hd, bs, seed=15)
    k, v = (torch.zeros(blocks, bs, nkv, hd, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    n = case.k.shape[0]
    k[-n:], v[-n:] = case.k, case.v
    tables = [[b + blocks - n if 0 <= b < n else b for b in row] for row in case.tables]
    got = ops.shared_prefix_attention(**case.args(k_cache=k, v_cache=v, block_tables=torch.tensor(tables, dtype=torch.int32, device=DEV)))
    case.check(got)
    assert torch.equal(got, ops.shared_prefix_attention(**case.args()))
