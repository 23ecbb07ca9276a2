"""ops.tree_attention on a B200 against its definition in 64 bits on the same bf16 inputs.

Tolerance, per element.  Rounding: the probabilities are rounded to bf16 for the second product, each by at most 2^-8 of itself, while their
sum is taken before: sum p (1 + e) v / sum p is off by at most 2^-8 A with A = sum p |v| / sum p, and the result's own rounding adds
2^-8 (|o| + that).  What is done in 32 bits: a score is a sum of head_dim <= 128 products, off by at most 128 * 2^-24 = 2^-17 of
S = scale * sum |q k|, which is about 11 for the draws here (standard deviations of 1.5 and 1), so by 2^-13, and p by that part of itself in the numerator and in
the sum below; exp2's argument and result add 2^-21 and less; sums over n keys add at most 2^-24 of A for every step of 64 keys (2^-15 at 32768).
Together below 2^-11 A, and 2^-10 A leaves room for scores of twice that size."""
import random

import pytest
import torch

import gpu_util
import step_util as ref

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
    """Sequences with prefixes[i] tokens before a tree of counts[i] nodes, in a cache whose other places hold NaN."""

    def __init__(self, prefixes, counts, nq=4, nkv=2, hd=128, bs=16, words=None, seed=0, std=1.5, extra_rows=0, reach=6):
        g = torch.Generator(device=DEV).manual_seed(seed)
        r = random.Random(seed)
        self.counts, self.lens = list(counts), [p + t for p, t in zip(prefixes, counts)]
        self.bs, self.scale = bs, hd ** -0.5
        width = max(1, -(-max(self.lens) // bs)) + 1
        used = sum(-(-n // bs) for n in self.lens)
        order = list(range(used + 5))
        r.shuffle(order)
        rows = []
        for n in self.lens:
            mine = [order.pop() for _ in range(-(-n // bs))]
            rows.append(mine + [r.choice((-1, 2 ** 31 - 1, -2 ** 31, 10 ** 6)) for _ in range(width - len(mine))])
        self.tables = torch.tensor(rows, dtype=torch.int32, device=DEV)
        shape = (used + 5, bs, nkv, hd)
        self.k = torch.full(shape, float("nan"), dtype=torch.bfloat16, device=DEV)
        self.v = torch.full(shape, float("nan"), dtype=torch.bfloat16, device=DEV)
        for b, n in enumerate(self.lens):
            slot = self.slots(b, range(n))
            for c in (self.k, self.v):
                c.view(-1, nkv, hd)[slot] = torch.empty(n, nkv, hd, dtype=torch.bfloat16, device=DEV).normal_(generator=g)
        tokens = sum(counts) + extra_rows
        self.q = torch.empty(tokens, nq, hd, dtype=torch.bfloat16, device=DEV).normal_(0, std, generator=g)
        words = words or max(1, -(-max(counts) // 64))
        self.mask = torch.cat([ref.trees(counts, words, seed, reach), torch.full((extra_rows, words), -1, dtype=torch.int64)]).to(DEV)
        self.max_q = max(counts)

    def slots(self, b, places):
        p = torch.tensor(list(places), dtype=torch.int64, device=DEV)
        return self.tables[b].long()[p // self.bs] * self.bs + p % self.bs

    def args(self):
        return (self.q, self.k, self.v, ref.cumulative(self.counts).to(DEV), torch.tensor(self.lens, dtype=torch.int32, device=DEV), self.tables, self.mask, max(1, self.max_q), self.scale)

    def check(self, ops, what=""):
        got = ops.tree_attention(*self.args())
        want, size = ref.tree_attention(self.q, self.k, self.v, self.counts, self.lens, self.tables, self.mask, self.scale)
        compare(got, want, size, what)
        return got


def compare(got, want, size, what=""):
    got = got.double()
    assert got.shape == want.shape
    nan = torch.isnan(want) | torch.isnan(size)
    inf = torch.isinf(want)
    assert torch.equal(torch.isnan(got), nan), f"{what}: NaN in {torch.isnan(got).sum().item()} places, expected {nan.sum().item()}"
    assert torch.equal(got[inf], want[inf]), f"{what}: infinities differ"
    fine = ~(nan | inf)
    err, bound = (got - want).abs()[fine], ((1 + HALF) * (HALF + FP32) * size + HALF * want.abs())[fine]
    if err.numel():
        worst = (err - bound).argmax()
        assert (err <= bound).all(), f"{what}: off by {err[worst].item():.3e}, bound {bound[worst].item():.3e}; {(err > bound).sum().item()} of {err.numel()} elements"


@pytest.mark.parametrize("nq, nkv", [(1, 1), (2, 2), (2, 1), (6, 2), (4, 1), (20, 4), (6, 1), (7, 1), (16, 2), (16, 1), (33, 1), (128, 1), (64, 8)])
@pytest.mark.parametrize("hd", [64, 128])
def test_head_layouts(ops, nq, nkv, hd):
    Case([70, 0, 129], [5, 9, 1], nq, nkv, hd, seed=nq * 31 + nkv).check(ops)


@pytest.mark.parametrize("bs", [16, 32, 48, 64, 80, 128, 256])
@pytest.mark.parametrize("hd", [64, 128])
def test_block_sizes(ops, bs, hd):
    """Tiles of keys that end inside a block, and blocks that end inside a tile."""
    Case([0, 1, bs - 1, bs, bs + 1, 3 * bs, 200], [3, 4, 5, 1, 7, 16, 13], bs=bs, hd=hd, seed=bs).check(ops)


@pytest.mark.parametrize("prefix", [0, 1, 15, 16, 17, 62, 63, 64, 65, 100, 127, 128, 129, 1000])
@pytest.mark.parametrize("nodes", [1, 2, 27, 63, 64, 65])
def test_contexts_and_trees_around_a_tile(ops, prefix, nodes):
    Case([prefix], [nodes], nq=8, nkv=2, seed=prefix * 100 + nodes).check(ops)


@pytest.mark.parametrize("nodes, words", [(1, 4), (100, 2), (128, 2), (129, 3), (200, 7), (700, 11)])
def test_large_trees_and_wide_masks(ops, nodes, words):
    Case([33, 0, 500], [nodes, 3, nodes // 2 + 1], nq=4, nkv=1, words=words, seed=nodes, reach=40).check(ops)


@pytest.mark.parametrize("nq, nkv, hd", [(8, 2, 128), (20, 4, 64), (16, 1, 128)])
def test_a_table_wider_than_the_contexts(ops, nq, nkv, hd):
    """Short contexts are one CTA's each where the table says that they are short, and are cut where it leaves room for longer ones."""
    c = Case([0, 60, 64, 301, 440, 3], [5, 64, 1, 20, 33, 7], nq, nkv, hd=hd, bs=16, seed=nq)
    c.check(ops, "narrow")
    c.tables = torch.cat([c.tables, torch.full((6, 500), -1, dtype=torch.int32, device=DEV)], 1)
    c.check(ops, "wide")


@pytest.mark.parametrize("max_q", [1, 9, 200])
def test_many_nodes_of_short_contexts(ops, max_q):
    """More nodes than the CTAs that walk side by side have rows for, whatever max_seqlen_q says."""
    c = Case([10, 0, 64], [200, 9, 130], nq=16, nkv=2, seed=26, reach=30)
    c.max_q = max_q
    c.check(ops)


def test_chains(ops):
    """Every node sees all nodes before it: what causal attention of the last tokens computes."""
    c = Case([300, 77], [64, 40], nq=8, nkv=2, seed=4)
    c.mask = ref.masks([(2 << i) - 1 for i in range(64)] + [(2 << i) - 1 for i in range(40)], 1).to(DEV)
    c.check(ops)


def test_ragged_batch(ops):
    r = random.Random(7)
    Case([r.randint(0, 900) for _ in range(37)], [r.randint(1, 33) for _ in range(37)], nq=10, nkv=2, bs=64, seed=7).check(ops)


def test_more_sequences_than_ctas(ops):
    r = random.Random(8)
    Case([r.randint(0, 150) for _ in range(400)], [r.randint(0, 6) for _ in range(400)], nq=4, nkv=2, bs=32, seed=8).check(ops)


@pytest.mark.parametrize("nq, nkv", [(8, 8), (64, 8), (5, 1)])
def test_a_long_context(ops, nq, nkv):
    Case([20011], [17], nq, nkv, bs=256, seed=9).check(ops)


def test_one_long_context_among_short_ones(ops):
    Case([5, 9000, 64, 3, 0, 700], [3, 40, 1, 64, 2, 9], nq=16, nkv=4, bs=128, seed=10).check(ops)


def test_nodes_that_see_nothing_and_sequences_without_a_context(ops):
    c = Case([0, 40, 0, 12], [6, 5, 3, 4], extra_rows=5, seed=11)
    c.mask[1] = 0      # before it there is nothing, and it sees no node: zeros
    c.mask[6 + 2] = 0  # sees the 40 tokens before the tree only
    c.mask[11:14] = 0
    c.lens[3] = 0      # a padded sequence
    got = c.check(ops)
    assert not got[1].any() and not got[11:].any()


def test_tokens_before_the_first_sequence_are_zero(ops):
    c = Case([20, 300], [4, 7], seed=27)
    q, k, v, cu, lens, tables, mask, max_q, scale = c.args()
    got = ops.tree_attention(q, k, v, cu[1:], lens[1:], tables[1:], mask, max_q, scale)
    want = ops.tree_attention(q, k, v, cu, lens, tables, mask, max_q, scale)
    assert not got[:4].any() and torch.equal(got[4:], want[4:])


@pytest.mark.parametrize("max_q", [2 ** 40, 2 ** 31 - 1, 10 ** 6])
def test_a_larger_max_seqlen_q(ops, max_q):
    c = Case([200, 30], [9, 4], seed=28)
    c.max_q = max_q
    c.check(ops)


def test_the_most_sequences_and_one_more(ops):
    Case([i % 40 for i in range(1024)], [1 + i % 3 for i in range(1024)], nq=2, nkv=1, hd=64, seed=29).check(ops)
    with pytest.raises(ValueError, match="1025 sequences"):
        ops.tree_attention(*Case([0] * 1025, [1] * 1025, nq=2, nkv=1, hd=64, seed=30).args())


@pytest.mark.parametrize("short", [-5, 0, 1, 3])
def test_a_context_shorter_than_its_tree(ops, short):
    c = Case([20, 30], [4, 4], seed=12)
    c.lens[0] = short
    assert not c.check(ops)[:4].any()


def test_no_sequences_and_no_tokens(ops):
    c = Case([20], [4], seed=13)
    q, k, v, cu, lens, tables, mask, max_q, scale = c.args()
    got = ops.tree_attention(q, k, v, cu[:1], lens[:0], tables[:0], mask, max_q, scale)
    assert got.shape == q.shape and not got.any()
    assert ops.tree_attention(q[:0], k, v, cu * 0, lens, tables, mask[:0], 0, scale).shape == (0, 4, 128)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), torch.finfo(torch.bfloat16).min, torch.finfo(torch.bfloat16).max])
@pytest.mark.parametrize("where", ["k", "v", "kv"])
def test_what_a_node_does_not_see_may_hold_anything(ops, bad, where):
    """Two branches; the second one's keys and values are bad.  The first one's results are what they are without them."""
    c = Case([70, 3], [6, 30], nq=8, nkv=2, seed=14)
    seen = [0b000001, 0b000011, 0b000101, 0b001011, 0b010101, 0b100011]
    c.mask[:6] = ref.masks(seen, 1).to(DEV)
    clean = ops.tree_attention(*c.args())
    slot = c.slots(0, [70 + 2])  # node 2: seen by itself and node 4
    if "k" in where:
        c.k.view(-1, 2, 128)[slot] = bad
    if "v" in where:
        c.v.view(-1, 2, 128)[slot, :, ::3] = bad
    got = ops.tree_attention(*c.args())
    rows = [0, 1, 3, 5] + list(range(6, 36))
    assert torch.equal(got[rows], clean[rows])


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("prefix", [70, 61, 3000])
def test_values_that_a_node_sees_reach_it(ops, prefix, bad):
    """Over contexts of one CTA and cut ones, in trees inside a tile and across two."""
    c = Case([prefix, 3], [6, 30], nq=8, nkv=2, seed=15)
    c.mask[:6] = ref.masks([0b000001, 0b000011, 0b000101, 0b001011, 0b010101, 0b100011], 1).to(DEV)
    c.v.view(-1, 2, 128)[c.slots(0, [prefix + 2]), :, ::3] = bad
    got = c.check(ops)
    assert not torch.isfinite(got[[2, 4]].float()[:, :, ::3]).any()


def test_a_nan_before_the_tree_reaches_every_node(ops):
    c = Case([400, 3], [6, 5], nq=8, nkv=2, seed=16)
    c.v.view(-1, 2, 128)[c.slots(0, [11]), 1, 5] = float("nan")
    c.check(ops)


@pytest.mark.parametrize("scale", [0.0, -0.09, 1e-30, 2.0])
def test_scales(ops, scale):
    c = Case([100, 0], [9, 20], nq=8, nkv=2, seed=17, std=0.5)
    c.scale = scale
    c.check(ops)


def test_growing_maxima(ops):
    """Scores that grow along the context: the running maximum moves in every tile."""
    c = Case([700], [20], nq=8, nkv=2, seed=18, std=0.2)
    place = c.slots(0, range(720))
    c.q += 1.0
    c.k.view(-1, 2, 128)[place] += torch.linspace(-2, 2, 720, device=DEV).view(-1, 1, 1).bfloat16()
    c.check(ops)


def test_bad_table_entries_stay_inside_the_cache(ops):
    """Entries that a context does use: the result is that of some block of the cache, and the other sequences are not touched."""
    c = Case([100, 100], [4, 4], seed=19)
    good = ops.tree_attention(*c.args())
    c.tables[0, :3] = torch.tensor([-7, 2 ** 31 - 1, 10 ** 7], dtype=torch.int32)
    got = ops.tree_attention(*c.args())
    assert torch.equal(got[4:], good[4:])


def test_q_as_a_view_of_the_projection(ops):
    c = Case([100, 31], [4, 9], nq=8, nkv=2, seed=20)
    want = ops.tree_attention(*c.args())
    wide = torch.full((13, 20, 128), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide[:, 4:12] = c.q
    c.q = wide[:, 4:12]
    assert torch.equal(ops.tree_attention(*c.args()), want)


def test_the_same_call_gives_the_same_bits(ops):
    c = Case([3000, 10, 800], [30, 64, 7], nq=32, nkv=8, bs=256, seed=21)
    first = ops.tree_attention(*c.args())
    assert all(torch.equal(ops.tree_attention(*c.args()), first) for _ in range(5))


def test_a_smaller_max_seqlen_q_changes_nothing_but_speed(ops):
    c = Case([100, 31], [100, 9], nq=8, nkv=2, seed=22)
    want = c.check(ops)
    c.max_q = 3
    compare(ops.tree_attention(*c.args()), *ref.tree_attention(c.q, c.k, c.v, c.counts, c.lens, c.tables, c.mask, c.scale))
    assert want is not None


def test_captured_calls_serve_later_batches_at_the_same_time(ops):
    """Two captured graphs with workspaces of their own, replayed side by side on two streams, with lengths that change."""
    cases = [Case([1500, 10, 800], [30, 64, 7], nq=32, nkv=8, bs=256, seed=23), Case([5000, 100, 0], [16, 16, 16], nq=8, nkv=4, bs=64, seed=24)]
    graphs, outs, args = [], [], []
    for c in cases:
        args.append(c.args())
        ops.tree_attention(*args[-1])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.tree_attention(*args[-1]))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for cut in (0, 3, 1):
        want = []
        for c, a in zip(cases, args):
            c.lens[0] -= cut * 64
            a[4].copy_(torch.tensor(c.lens, dtype=torch.int32))
            want.append(ref.tree_attention(c.q, c.k, c.v, c.counts, c.lens, c.tables, c.mask, c.scale))
        torch.cuda.synchronize()
        for _ in range(10):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for out, (w, s) in zip(outs, want):
            compare(out, w, s, f"cut {cut}")


def test_on_another_stream(ops):
    c = Case([100, 31], [4, 9], nq=8, nkv=2, seed=25)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = ops.tree_attention(*c.args())
    stream.synchronize()
    compare(got, *ref.tree_attention(c.q, c.k, c.v, c.counts, c.lens, c.tables, c.mask, c.scale))


def test_places_past_32_bits_of_elements(ops):
    """A cache of more than 2^31 elements, read at its end."""
    free, _ = torch.cuda.mem_get_info()
    blocks, bs, nkv, hd = 9000, 256, 8, 128
    if free < 3 * 2 * blocks * bs * nkv * hd:
        pytest.skip("not enough memory")
    k = torch.empty(blocks, bs, nkv, hd, dtype=torch.bfloat16, device=DEV)
    v = torch.empty(blocks, bs, nkv, hd, dtype=torch.bfloat16, device=DEV)
    assert k.numel() > 2 ** 31
    mine = [8999, 8990, 3, 8995]
    for b in mine:
        k[b].normal_()
        v[b].normal_()
    q = torch.empty(9, 16, hd, dtype=torch.bfloat16, device=DEV).normal_()
    tables = torch.tensor([mine], dtype=torch.int32, device=DEV)
    mask = ref.trees([9], 1, 1)
    got = ops.tree_attention(q, k, v, ref.cumulative([9]).to(DEV), torch.tensor([900], dtype=torch.int32, device=DEV), tables, mask.to(DEV), 9, 0.09)
    compare(got, *ref.tree_attention(q, k, v, [9], [900], tables, mask, 0.09))
