"""Timed cases of the operators of a beam-search step, through the calls a serving program makes.

  prefix   ops.shared_prefix_attention: decode attention of sequences that share the beginning of their contexts
  select   ops.beam_select: the best continuations of each request, over its beams and the vocabulary
  reorder  ops.reorder_beams: block tables, cache and token histories follow the beams that were selected

The sizes are those of the models and limits of engine/model_runner.py (8 KV heads of 128, 16 to 64 query heads, 28 and 36
layers, 151936 tokens of vocabulary, blocks of 256, 512 sequences), and generic ones around them.
"""
import math
import random
from collections import Counter

import torch

own = False

VOCAB = 151936


# ---- the cases -------------------------------------------------------------------------------------------------
def _prefix(name, groups, size, ragged, longest, shortest, tail, nq, nkv, hd, block):
    """groups of `size` sequences (1..size where ragged) behind shortest..longest common tokens, each with 1..tail tokens of its own."""
    return dict(name=name, kind="prefix", groups=groups, size=size, ragged=ragged, longest=longest, shortest=shortest, tail=tail, nq=nq, nkv=nkv, hd=hd, block=block)


def _select(name, requests, beams, picks, vocab, dtype, masked, finished):
    """picks continuations for each request of `beams` beams; a share `masked` of the vocabulary forbidden, a share of the beams at their end."""
    return dict(name=name, kind="select", requests=requests, beams=beams, picks=picks, vocab=vocab, dtype=dtype, masked=masked, finished=finished)


def _reorder(name, requests, beams, longest, shortest, steps, block, layers, nkv, width):
    """requests with prompts of shortest..longest tokens whose beams have come apart over the last `steps`; histories of `width` tokens."""
    return dict(name=name, kind="reorder", requests=requests, beams=beams, longest=longest, shortest=shortest, steps=steps, block=block, layers=layers, nkv=nkv, width=width)


def listed():
    return [
        # one user, four beams behind a short prompt: launches and latency
        _prefix("prefix_one", 1, 4, False, 300, 300, 40, 16, 8, 128, 256),
        # a server that searches with eight beams for each of eight users
        _prefix("prefix_beams", 8, 8, False, 4096, 2000, 512, 32, 8, 128, 256),
        # beams and batches of all sizes, odd heads and small blocks
        _prefix("prefix_ragged", 9, 13, True, 3001, 1, 700, 20, 4, 64, 16),
        # a full server whose users all talk to it behind one long system prompt
        _prefix("prefix_system", 1, 256, False, 8192, 8192, 1500, 64, 8, 128, 256),
        # one user with four beams
        _select("select_one", 1, 4, 4, VOCAB, "bf16", 0.0, 0.0),
        # as many rows as a server has sequences
        _select("select_batch", 64, 8, 8, VOCAB, "bf16", 0.0, 0.0),
        # logits in 32 bits, an odd vocabulary, odd numbers of beams and picks
        _select("select_fp32", 33, 3, 7, 50257, "fp32", 0.0, 0.1),
        # wide beams whose grammar forbids most tokens, some of them at their end
        _select("select_grammar", 5, 32, 64, VOCAB, "bf16", 0.9, 0.3),
        # one user with four beams, blocks of 256 tokens in all layers
        _reorder("reorder_one", 1, 4, 300, 300, 40, 256, 28, 8, 4096),
        # a full server of short blocks, one rank of eight
        _reorder("reorder_batch", 64, 8, 600, 100, 60, 16, 36, 1, 1024),
        # long documents
        _reorder("reorder_long", 2, 5, 20001, 15000, 300, 64, 28, 2, 32768),
        # wide beams, odd sizes
        _reorder("reorder_wide", 7, 29, 999, 1, 130, 48, 9, 3, 1200),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("prefix", "select", "reorder"))
    if kind == "prefix":
        while True:
            size, groups = _log(rng, 1, 256), _log(rng, 1, 64)
            longest, tail = _log(rng, 1, 16384), _log(rng, 1, 2000)
            nkv, hd = rng.choice((1, 2, 4, 8, 8)), rng.choice((64, 128, 128))
            group = rng.choice((1, 2, 3, 4, 4, 5, 8, 8))
            kv = (groups * longest + groups * size * tail) * nkv * hd
            if groups * size <= 512 and kv <= (8192 + 256 * 1500) * 8 * 128 and size * groups * (longest + tail) * group * nkv * hd <= 256 * 9000 * 64 * 128:
                break
        return _prefix("", groups, size, rng.random() < 0.5, longest, rng.randint(1, longest), tail, group * nkv, nkv, hd, rng.choice((16, 32, 48, 64, 128, 256)))
    if kind == "select":
        vocab, dtype = rng.choice((VOCAB, VOCAB, 50257, _log(rng, 1000, 160000))), rng.choice(("bf16", "bf16", "fp32"))
        rows, beams = _log(rng, 1, 240 if dtype == "fp32" else 480), _log(rng, 1, 32)
        picks = rng.choice((beams, beams, min(64, 2 * beams), rng.randint(1, 64)))
        return _select("", max(1, rows // beams), beams, picks, vocab, dtype, rng.choice((0.0, 0.0, 0.5, 0.999)), rng.choice((0.0, 0.0, 0.3)))
    while True:
        requests, beams = _log(rng, 1, 128), _log(rng, 1, 32)
        longest, steps = _log(rng, 1, 20000), _log(rng, 1, 400)
        block, layers, nkv = rng.choice((16, 32, 48, 64, 128, 256)), _log(rng, 1, 40), rng.choice((1, 2, 3, 4, 8))
        blocks = requests * (longest // block + beams * (2 + steps // block))
        if requests * beams <= 512 and blocks * block * layers * nkv * 512 <= 1 << 30 and requests * beams * longest <= 1 << 19:
            break
    return _reorder("", requests, beams, longest, rng.randint(1, longest), steps, block, layers, nkv, longest + steps + rng.randint(1, 2000))


# ---- the inputs --------------------------------------------------------------------------------------------------
def _lens(what, n, longest, shortest):
    """Lengths from shortest to longest; they belong to the case, whatever the inputs' seed."""
    r = random.Random(f"{what} {n} {longest} {shortest}")
    out = [r.randint(shortest, longest) for _ in range(n)]
    out[r.randrange(n)] = longest
    return out


def _prefix_lens(case):
    """Sequences of each group, its common tokens, and each sequence's length."""
    sizes = _lens("sizes", case["groups"], case["size"], 1) if case["ragged"] else [case["size"]] * case["groups"]
    common = _lens("common", case["groups"], case["longest"], case["shortest"])
    tails = _lens("tails", sum(sizes), case["tail"], 1)
    of = [g for g, size in enumerate(sizes) for _ in range(size)]
    return sizes, common, [common[g] + t for g, t in zip(of, tails)]


def _cumulative(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _gpu(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


class State:
    def __init__(self, **kw):
        self.__dict__.update(kw)


def _prepare_prefix(case, seed):
    sizes, common, lens = _prefix_lens(case)
    r, g = random.Random(seed), _gpu(seed)
    bs, nkv, hd = case["block"], case["nkv"], case["hd"]
    shared = [c // bs for c in common]  # full blocks of common tokens; what is left of them is in each sequence's own
    width = max(-(-n // bs) for n in lens)
    blocks, at = sum(shared) + 3, 0
    for s, size in zip(shared, sizes):
        blocks += sum(-(-n // bs) - s for n in lens[at:at + size])
        at += size
    order = list(range(blocks))
    r.shuffle(order)
    rows, at = [], 0
    for s, size in zip(shared, sizes):
        first = [order.pop() for _ in range(s)]
        for n in lens[at:at + size]:
            mine = first + [order.pop() for _ in range(-(-n // bs) - s)]
            rows.append(mine + [-1] * (width - len(mine)))
        at += size
    k = torch.empty(blocks, bs, nkv, hd, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    v = torch.empty(blocks, bs, nkv, hd, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    q = torch.empty(len(lens), case["nq"], hd, dtype=torch.bfloat16, device="cuda").normal_(0, 1.5, generator=g)
    return State(kind="prefix", q=q, k=k, v=v, cu=_int32(_cumulative(sizes)), prefix=_int32([s * bs for s in shared]), lens=_int32(lens), tables=_int32(rows), largest=max(sizes),
                 scale=hd ** -0.5, block=bs, sizes=sizes, host_prefix=[s * bs for s in shared], host_lens=lens)


def _prepare_select(case, seed):
    n, b, v = case["requests"], case["beams"], case["vocab"]
    g = _gpu(seed)
    dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    logits = torch.empty(n * b, v, dtype=dtype, device="cuda").normal_(0, 3, generator=g)
    if case["masked"]:
        logits.masked_fill_(torch.empty(n * b, v, device="cuda").uniform_(generator=g) < case["masked"], float("-inf"))
    scores = torch.empty(n, b, device="cuda").uniform_(-14, -10, generator=g)
    finished = None
    if case["finished"]:
        finished = torch.empty(n, b, device="cuda").uniform_(generator=g) < case["finished"]
        scores[:, b // 2:].masked_fill_(torch.empty(n, b - b // 2, device="cuda").uniform_(generator=g) < 0.1, float("-inf"))  # beams that a request has not got
    return State(kind="select", logits=logits, scores=scores, picks=case["picks"], finished=finished, eos=v // 2)


def _tables(case, seed):
    """Tables of beams that have come apart: beam i shares what it has in common with an earlier one, as far as it fills blocks."""
    r = random.Random(seed)
    b, bs, steps = case["beams"], case["block"], case["steps"]
    prompts = _lens("prompts", case["requests"], case["longest"], case["shortest"])
    rows, lens, number = [], [], 0
    for p in prompts:
        mine, longs = [], []
        for i in range(b):
            n = p + steps if r.random() < 0.8 else p + r.randint(0, steps)  # some have ended early
            table = []
            if i > 0:
                a = r.randrange(i)
                table = mine[a][:min(r.randint(p, p + steps), n, longs[a]) // bs]
            fresh = -(-n // bs) - len(table)
            table = table + list(range(number, number + fresh))
            number += fresh
            mine.append(table)
            longs.append(n)
        rows += mine
        lens += longs
    return rows, lens, [p // bs for p in prompts], number


def _prepare_reorder(case, seed):
    n, b, bs = case["requests"], case["beams"], case["block"]
    rows, lens, first, number = _tables(case, f"{sorted(case.items())}")
    r, g = random.Random(seed), _gpu(seed)
    blocks = number + n * b + 5
    order = list(range(blocks))
    r.shuffle(order)
    width = max(-(-x // bs) for x in lens) + 2
    rows = [[order[x] for x in row] + [-1] * (width - len(row)) for row in rows]
    free = order[number:]
    parents, tokens = [], []
    for _ in range(n):
        # good beams have several children, bad ones none
        ranks = [min(b - 1, int(r.expovariate(2.0) * b)) for _ in range(b)]
        parents.append([-1 if b > 2 and r.random() < 0.02 else x for x in ranks])
        tokens.append([-1 if r.random() < 0.05 else r.randrange(VOCAB) for _ in range(b)])
    cache = torch.empty(2, case["layers"], blocks, bs, case["nkv"], 128, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    history = torch.randint(0, VOCAB, (n * b, case["width"]), device="cuda", generator=g)
    return State(kind="reorder", parents=_int32(parents), tables=_int32(rows), lens=_int32(lens), free=_int32(free + [-1] * number), num_free=_int32([len(free)]), cache=cache,
                 first=_int32(first), history=history, history_lens=_int32([min(x + 1, case["width"]) for x in lens]), tokens=torch.tensor(tokens, device="cuda"))


def _package():
    import __graft_entry__
    package = __graft_entry__.load_package()
    from nanovllm_b200 import ops, runtime
    if runtime._RUNTIME is None:
        package.init_runtime(max_tokens=16384, hidden=4096)
    return ops


_PREPARE = {"prefix": _prepare_prefix, "select": _prepare_select, "reorder": _prepare_reorder}


def prepare(case, seed):
    state = _PREPARE[case["kind"]](case, seed)
    if own:
        state.ops = _package()
    return state


# ---- the plain forms -----------------------------------------------------------------------------------------------
def _plain_prefix(s):
    nkv, hd = s.k.shape[2:]
    nq = s.q.shape[1]
    outs, at = [], 0
    for size, p in zip(s.sizes, s.host_prefix):  # (groups differ in every length)
        rows, width = slice(at, at + size), max(s.host_lens[at:at + size]) - p
        q = s.q[rows].float().view(size, nkv, nq // nkv, hd).transpose(0, 1)  # [nkv, size, heads of a group, hd]
        front = s.tables[at, :p // s.block].long()
        k, v = (x[front].reshape(p, nkv, hd).float().transpose(0, 1) for x in (s.k, s.v))  # [nkv, p, hd]
        place = p + torch.arange(width, device=q.device)
        slot = s.tables[rows].long().gather(1, (place // s.block).expand(size, width)).clamp(min=0) * s.block + place % s.block
        tail_k, tail_v = (x.view(-1, nkv, hd)[slot].float().permute(2, 0, 1, 3) for x in (s.k, s.v))  # [nkv, size, width, hd]
        back = (q @ tail_k.transpose(-1, -2) * s.scale).masked_fill_((place >= s.lens[rows].unsqueeze(1)).unsqueeze(1), float("-inf"))
        tail_v = tail_v.masked_fill((place >= s.lens[rows].unsqueeze(1)).unsqueeze(-1), 0.0)
        score = torch.cat([(q.reshape(nkv, -1, hd) @ k.transpose(-1, -2) * s.scale).view(nkv, size, nq // nkv, p), back], -1)
        e = torch.exp(score - score.amax(-1, keepdim=True))
        o = (e[..., :p].reshape(nkv, size * (nq // nkv), p) @ v).view(q.shape) + e[..., p:] @ tail_v
        outs.append((o / e.sum(-1, keepdim=True)).transpose(0, 1).reshape(size, nq, hd).to(torch.bfloat16))
        at += size
    return torch.cat(outs)


def _plain_select(s):
    n, b = s.scores.shape
    v, dev = s.logits.shape[1], s.logits.device
    x = s.logits.double()
    top = x.amax(-1, keepdim=True)
    total = top + torch.exp(x - top).sum(-1, keepdim=True).log()  # NaN where a beam may go nowhere, which is sorted out below
    # each beam's best tokens, the lowest of equal ones first: a key of the logit's order and the token's number
    k = min(s.picks, v)
    bits = (s.logits.float() + 0.0).view(torch.int32).long()  # (-0 equals 0)
    rank = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    key = (rank << 32) + (v - 1 - torch.arange(v, device=dev))
    token = torch.topk(key, k, dim=-1).indices.sort(-1).values
    score = s.scores.double().view(-1, 1) + (x.gather(1, token) - total)
    score = torch.where(torch.isnan(score), float("-inf"), score)
    if s.finished is not None:  # these go on as they are: one continuation, without a token
        ended = s.finished.view(-1, 1)
        alone = torch.where(torch.arange(k, device=dev) == 0, s.scores.double().view(-1, 1), float("-inf"))
        score, token = torch.where(ended, alone, score), torch.where(ended, -1, token)
    score, token = score.view(n, b * k), token.view(n, b * k)
    if b * k < s.picks:
        more = s.picks - b * k
        score = torch.cat([score, torch.full((n, more), float("-inf"), dtype=torch.float64, device=dev)], 1)
        token = torch.cat([token, torch.full((n, more), -1, device=dev)], 1)
    score, order = torch.sort(score, dim=-1, descending=True, stable=True)
    score, order = score[:, :s.picks], order[:, :s.picks]
    there = score > float("-inf")
    parent, token = torch.where(there, order // k, -1), torch.where(there, token.gather(1, order), -1)
    finished = there & (token == s.eos)
    if s.finished is not None:
        finished |= there & s.finished.gather(1, parent.clamp(min=0))
    return score.float(), parent.int(), token, finished


def _plain_reorder(s):
    n, b = s.parents.shape
    width, dev = s.tables.shape[1], s.tables.device
    planes, blocks, bs = s.cache.shape[0] * s.cache.shape[1], s.cache.shape[2], s.cache.shape[3]
    old, lens, parent, first = s.tables.view(n, b, width).long(), s.lens.view(n, b).long(), s.parents.long(), s.first.long().unsqueeze(1)
    column = torch.arange(width, device=dev)
    alive, p = parent >= 0, parent.clamp(min=0)
    new_lens = torch.where(alive, lens.gather(1, p), 0)
    deep = p.unsqueeze(-1).expand(n, b, width)
    new = torch.where(column < ((new_lens + bs - 1) // bs).unsqueeze(-1), old.gather(1, deep), -1)
    # the open block stays with the first row that has it; the others get a copy of it
    open_at = new_lens // bs
    in_column = new.gather(2, open_at.clamp(max=width - 1).unsqueeze(1).expand(n, b, b))  # [request, row, whose open column]
    mine = torch.where(new_lens % bs > 0, in_column.diagonal(dim1=1, dim2=2), -1)
    keeper = (in_column == mine.unsqueeze(1)).float().argmax(1)
    copied = (mine >= 0) & (keeper != torch.arange(b, device=dev))
    held = torch.where(copied.unsqueeze(-1) & (column == open_at.unsqueeze(-1)), -1, new)
    # blocks that no row holds any more, by column and row, each once
    given = (column < ((lens + bs - 1) // bs).unsqueeze(-1)) & (column >= torch.minimum(first, lens // bs).unsqueeze(-1)) & (old >= 0)
    wanted = (old.unsqueeze(2) == held.unsqueeze(1)).any(2)
    earlier = torch.arange(b, device=dev).unsqueeze(0) < torch.arange(b, device=dev).unsqueeze(1)  # [row, another before it]
    again = ((old.unsqueeze(2) == old.unsqueeze(1)) & given.unsqueeze(1) & earlier.unsqueeze(-1)).any(2)
    back = (given & ~wanted & ~again).transpose(1, 2).reshape(-1)
    place = back.long().cumsum(0)
    returned = torch.full((back.numel() + 1,), -1, device=dev).scatter_(0, torch.where(back, place - 1, back.numel()), old.transpose(1, 2).reshape(-1))
    # copies take their blocks from the top of the stack
    free = s.num_free.long().clamp(0, s.free.numel())
    top = free + place[-1]
    turn = copied.view(-1).long().cumsum(0).view(n, b) - 1
    at = top - 1 - turn
    block = torch.where(at < free, s.free.long()[at.clamp(0, s.free.numel() - 1)], returned[(at - free).clamp(0, back.numel())])
    served = copied & (at >= 0)
    tables = torch.where(served.unsqueeze(-1) & (column == open_at.unsqueeze(-1)), block.unsqueeze(-1), held)
    tokens_in_open = new_lens - open_at * bs
    new_lens = torch.where(copied & ~served, open_at * bs, new_lens)
    left = (top - copied.sum()).clamp(min=0, max=s.free.numel())
    i = torch.arange(s.free.numel(), device=dev)
    s.free.copy_(torch.where((i >= free) & (i < left), returned[(i - free).clamp(0, back.numel())], s.free))
    # the copied tokens in all planes
    inside = torch.arange(bs, device=dev)
    request, row, token = torch.nonzero(served.unsqueeze(-1) & (inside < tokens_in_open.unsqueeze(-1)), as_tuple=True)
    flat = s.cache.view(planes, blocks * bs, -1)
    flat[:, block[request, row] * bs + token] = flat[:, mine[request, row] * bs + token]
    # histories, with the token that each row has been given
    wide = s.history.shape[1]
    line = (torch.arange(n, device=dev).unsqueeze(1) * b + p).view(-1)
    said = torch.where(alive.view(-1), s.history_lens.long()[line], 0).unsqueeze(1)
    token, spot = s.tokens.view(-1, 1), torch.arange(wide, device=dev)
    says = alive.view(-1, 1) & (token >= 0) & (said < wide)
    history = torch.where(spot < said, s.history[line], torch.where(says & (spot == said), token, -1))
    return tables.view(n * b, width).int(), new_lens.view(-1).int(), left.int(), s.free, s.cache, history, (said + says).view(-1).int()


# ---- the calls -----------------------------------------------------------------------------------------------------
_PLAIN = {"prefix": _plain_prefix, "select": _plain_select, "reorder": _plain_reorder}


def run(state):
    s = state
    if not own:
        return _PLAIN[s.kind](s)
    if s.kind == "prefix":
        return s.ops.shared_prefix_attention(s.q, s.k, s.v, s.cu, s.prefix, s.lens, s.tables, s.largest, s.scale)
    if s.kind == "select":
        return tuple(s.ops.beam_select(s.logits, s.scores, s.picks, finished=s.finished, eos_token=s.eos))
    r = s.ops.reorder_beams(s.parents, s.tables, s.lens, s.free, s.num_free, s.cache, first_blocks=s.first, history=s.history, history_lens=s.history_lens, tokens=s.tokens)
    return r.block_tables, r.context_lens, r.num_free, s.free, s.cache, r.history, r.history_lens


# ---- what a pass cannot do without -------------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "prefix":
        sizes, common, lens = _prefix_lens(case)
        bs, row = case["block"], 4 * case["nkv"] * case["hd"]
        shared, at, tails = [c // bs * bs for c in common], 0, 0
        for s, size in zip(shared, sizes):
            tails += sum(lens[at:at + size]) - s * size
            at += size
        return {"bytes": row * (sum(shared) + tails) + 4 * len(lens) * case["nq"] * case["hd"] + 4 * (sum(shared) + tails) // bs, "flops": 4 * sum(lens) * case["nq"] * case["hd"]}
    if case["kind"] == "select":
        rows = case["requests"] * case["beams"]
        return {"bytes": (2 if case["dtype"] == "bf16" else 4) * rows * case["vocab"] + 17 * case["requests"] * case["picks"] + 5 * rows, "flops": 4 * rows * case["vocab"]}
    rows, lens, _, _ = _tables(case, f"{sorted(case.items())}")
    n, bs = case["requests"] * case["beams"], case["block"]
    # (a beam in three or so has lost its place to another one's child, which then needs a copy of half a block)
    return {"bytes": 8 * sum(len(r) for r in rows) + 8 * sum(lens) + 8 * n * case["width"] + n // 3 * bs * case["layers"] * case["nkv"] * 512, "flops": n * case["width"]}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
def _exact_prefix(s):
    n, nq, hd = s.q.shape
    nkv = s.k.shape[2]
    out = torch.empty(n, nq, hd, dtype=torch.float64, device="cuda")
    for i, length in enumerate(s.host_lens):
        place = torch.arange(length, device="cuda")
        slot = s.tables[i].long()[place // s.block] * s.block + place % s.block
        k, v = s.k.view(-1, nkv, hd)[slot].double(), s.v.view(-1, nkv, hd)[slot].double()
        p = torch.softmax(torch.einsum("hgd,thd->hgt", s.q[i].double().view(nkv, nq // nkv, hd), k) * s.scale, -1)
        out[i] = torch.einsum("hgt,thd->hgd", p, v).reshape(nq, hd)
    return out


def _exact_select(s):
    n, b = s.scores.shape
    v, picks = s.logits.shape[1], s.picks
    scores = torch.full((n, picks), float("-inf"), dtype=torch.float64, device="cuda")
    parents = torch.full((n, picks), -1, dtype=torch.int32, device="cuda")
    tokens = torch.full((n, picks), -1, dtype=torch.int64, device="cuda")
    ended = torch.zeros(n, picks, dtype=torch.bool, device="cuda")
    for i in range(n):
        x = torch.log_softmax(s.logits[i * b:(i + 1) * b].double(), -1) + s.scores[i].double().unsqueeze(1)
        x = torch.nan_to_num(x, nan=float("-inf"), neginf=float("-inf"))
        done = s.finished[i].tolist() if s.finished is not None else [False] * b
        for j in range(b):
            if done[j]:
                x[j] = float("-inf")
                x[j, 0] = s.scores[i, j].double()
        values, at = torch.sort(x.view(-1), descending=True, stable=True)
        for k, (value, place) in enumerate(zip(values[:picks].tolist(), at[:picks].tolist())):
            if value > float("-inf"):
                j, token = divmod(place, v)
                scores[i, k], parents[i, k], tokens[i, k], ended[i, k] = value, j, -1 if done[j] else token, done[j] or token == s.eos
    return scores, parents, tokens, ended


def _exact_reorder(s):
    """A request at a time with a count of each block's holders, as a block manager on the host does it."""
    n, b = s.parents.shape
    bs, wide, width = s.cache.shape[3], s.history.shape[1], s.tables.shape[1]
    tables, lens, free, height = s.tables.tolist(), s.lens.tolist(), s.free.tolist(), s.num_free.item()
    parents, first, tokens = s.parents.tolist(), s.first.tolist(), s.tokens.tolist()
    stack, plans, new_tables, new_lens = free[:height], [], [], []
    for i in range(n):
        old = [tables[i * b + q][:-(-lens[i * b + q] // bs)] for q in range(b)]
        new, taken = [], []
        holders, opened = Counter(), set()
        for c in range(b):
            q = parents[i][c]
            length = lens[i * b + q] if q >= 0 else 0
            row = list(old[q]) if q >= 0 else []
            copy = None
            if length % bs and row[-1] in opened:
                copy, row[-1] = (row[-1], length % bs), None
            elif length % bs:
                opened.add(row[-1])
            holders.update(x for x in row if x is not None)
            new.append(row)
            new_lens.append(length)
            taken.append(copy)
        gone = set()
        for j in range(max(map(len, old))):
            for q in range(b):
                if first[i] <= j < len(old[q]) and not holders[old[q][j]] and old[q][j] not in gone:
                    gone.add(old[q][j])
                    stack.append(old[q][j])
        new_tables += new
        plans += taken
    cache = s.cache.view(-1, *s.cache.shape[2:])
    moves = []
    for row, copy in enumerate(plans):
        if copy:
            new_tables[row][-1] = stack.pop()
            moves.append((copy[0], new_tables[row][-1], copy[1]))
    for src, dst, count in moves:
        cache[:, dst, :count] = cache[:, src, :count]
    free[height:max(height, len(stack))] = stack[height:]
    history, said = torch.full_like(s.history, -1), []
    for row in range(n * b):
        q = parents[row // b][row % b]
        length = 0
        if q >= 0:
            length = s.history_lens[row // b * b + q].item()
            history[row, :length] = s.history[row // b * b + q, :length]
            if tokens[row // b][row % b] >= 0 and length < wide:
                history[row, length] = tokens[row // b][row % b]
                length += 1
        said.append(length)
    return _int32([r + [-1] * (width - len(r)) for r in new_tables]), _int32(new_lens), _int32([len(stack)]), _int32(free), s.cache, history, _int32(said)


def exact(case, seed):
    state = _PREPARE[case["kind"]](case, seed)
    return {"prefix": _exact_prefix, "select": _exact_select, "reorder": _exact_reorder}[case["kind"]](state)
