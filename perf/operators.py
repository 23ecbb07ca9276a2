"""Timed cases of the operators around a verification step of drafted tokens, through the calls a serving program makes.

  inputs   ops.batch_inputs: block tables, positions and slots of a batch, from the requests' lengths and a stack of free blocks
  tree     ops.tree_attention: attention of a tree of drafted tokens per sequence over the paged cache
  logits   ops.adjust_logits: penalties for repeated tokens, biases and grammar masks on logits

The sizes are those of the models and limits of engine/model_runner.py (8 KV heads of 128, 16 to 64 query heads, 151936
tokens of vocabulary, blocks of 256, steps of 16384 tokens, 512 sequences), and generic ones around them.
"""
import math
import random

import torch

own = False

VOCAB = 151936
HEADS = ((16, 8), (32, 8), (64, 8))


# ---- the cases -------------------------------------------------------------------------------------------------
def _inputs(name, rows, longest, shortest, block, add, prompt=0, prompts=0, done=0.0, tree=False):
    """rows requests with shortest..longest tokens in the cache, each to get `add` more; the last `prompts` of them are new
    and get `prompt` tokens; a share `done` of the others is finished and gives its blocks back."""
    return dict(name=name, kind="inputs", rows=rows, longest=longest, shortest=shortest, block=block, add=add, prompt=prompt,
                prompts=prompts, done=done, tree=tree)


def _tree(name, seqs, longest, shortest, nodes, ragged, nq, nkv, hd, block):
    """seqs sequences of shortest..longest cached tokens and trees of `nodes` drafted tokens (1..nodes where ragged)."""
    return dict(name=name, kind="tree", seqs=seqs, longest=longest, shortest=shortest, nodes=nodes, ragged=ragged, nq=nq, nkv=nkv,
                hd=hd, block=block)


def _logits(name, seqs, nodes, vocab, history, dtype, penalties, bias, mask):
    """seqs requests of history/2..history tokens, one row of logits each, or one per node of a tree of drafted tokens."""
    return dict(name=name, kind="logits", seqs=seqs, nodes=nodes, vocab=vocab, history=history, dtype=dtype, penalties=penalties,
                bias=bias, mask=mask)


def listed():
    return [
        # one user chatting: a single decode step's inputs
        _inputs("inputs_one", 1, 300, 300, 256, 1),
        # a full server of short-block tables: 512 requests take a token each, one in ten has finished and gives its blocks back
        _inputs("inputs_full", 512, 4096, 1, 16, 1, done=0.1),
        # a step of 16384 tokens: running requests and long prompts in one batch
        _inputs("inputs_prompts", 131, 4096, 40, 256, 1, prompt=5417, prompts=3),
        # trees of drafted tokens: positions follow the depth in the tree
        _inputs("inputs_trees", 37, 2000, 100, 64, 16, tree=True),
        # one user, a short context and a few drafted tokens: launches and latency
        _tree("tree_one", 1, 300, 300, 5, False, 16, 8, 128, 256),
        # one user, a long context and a wide tree of a large model
        _tree("tree_long", 1, 32768, 32768, 64, False, 64, 8, 128, 256),
        # a lightly loaded server: contexts of all lengths, trees of all sizes, odd heads and small blocks
        _tree("tree_ragged", 21, 3001, 1, 27, True, 20, 4, 64, 16),
        # a busy server: 64 sequences of 4096 tokens and trees of 32
        _tree("tree_many", 64, 4096, 4000, 32, False, 32, 8, 128, 256),
        # one user with penalties
        _logits("logits_one", 1, 0, VOCAB, 1024, "bf16", True, 8, False),
        # a server's batch with all rules
        _logits("logits_batch", 64, 0, VOCAB, 4096, "bf16", True, 300, True),
        # logits in 32 bits, an odd vocabulary, long histories
        _logits("logits_fp32", 33, 0, 50257, 30001, "fp32", True, 0, False),
        # verification of trees: every node has a grammar state and the drafted tokens before it
        _logits("logits_trees", 32, 16, VOCAB, 2048, "bf16", True, 16, True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("inputs", "tree", "tree", "logits"))
    if kind == "inputs":
        rows, block = _log(rng, 1, 512), rng.choice((16, 32, 64, 128, 256))
        longest = _log(rng, 2, 4096)
        tree = rng.random() < 0.3
        add = _log(rng, 1, max(1, min(32, 16384 // rows))) if tree else rng.choice((1, 1, 1 + _log(rng, 1, max(1, min(64, 16384 // rows - 1)))))
        prompts = 0 if tree or rows == 1 else rng.choice((0, min(rows - 1, _log(rng, 1, 8))))
        prompt = _log(rng, 1, max(1, (16384 - add * rows) // max(1, prompts))) if prompts else 0
        prompt = max(0, min(prompt, (16384 - add * (rows - prompts)) // max(1, prompts)))
        return _inputs("", rows, longest, rng.randint(1, longest), block, add, prompt=prompt, prompts=prompts if prompt else 0,
                       done=rng.choice((0.0, 0.0, 0.1, 0.5)), tree=tree)
    if kind == "tree":
        while True:
            seqs, longest, nodes = _log(rng, 1, 64), _log(rng, 1, 32768), _log(rng, 1, 64)
            nkv, hd = rng.choice((1, 2, 4, 8, 8)), rng.choice((64, 128, 128))
            group = rng.choice((1, 2, 2, 3, 4, 4, 5, 7, 8))
            pairs = seqs * (longest + nodes) * nkv * hd
            if pairs <= 64 * 4128 * 8 * 128 and pairs * nodes * group <= 64 * 4096 * 8 * 128 * 32 * 4:
                break
        return _tree("", seqs, longest, rng.randint(1, longest), nodes, rng.random() < 0.5, group * nkv, nkv, hd, rng.choice((16, 32, 64, 128, 256, 48)))
    vocab = rng.choice((VOCAB, VOCAB, 50257, _log(rng, 1000, 160000)))
    nodes = rng.choice((0, 0, _log(rng, 1, 32)))
    rows = _log(rng, 1, 512)
    seqs = max(1, rows // max(1, nodes))
    history = _log(rng, 1, 32768)
    history = min(history, 1 << 21 if seqs == 1 else (1 << 21) // seqs)
    dtype = rng.choice(("bf16", "bf16", "fp32"))
    if dtype == "fp32" or vocab > VOCAB:
        seqs = max(1, seqs // 2)
    return _logits("", seqs, nodes, vocab, max(1, history), dtype, rng.random() < 0.8, rng.choice((0, 0, _log(rng, 1, 300))), rng.random() < 0.5)


# ---- the inputs --------------------------------------------------------------------------------------------------
def _lens(seed, n, longest, shortest):
    """Lengths from shortest to longest; they belong to the case, whatever the inputs' seed."""
    r = random.Random(f"{seed} {n} {longest} {shortest}")
    out = [r.randint(shortest, longest) for _ in range(n)]
    out[r.randrange(n)] = longest
    return out


def _row_lens(case):
    """What each row of an "inputs" case has in the cache and what it is to have."""
    n, new = case["rows"], case["prompts"]
    cached = _lens("rows", n, case["longest"], case["shortest"])
    for i in range(n - new, n):
        cached[i] = 0
    r = random.Random(f"done {n}")
    want = []
    for i, c in enumerate(cached):
        if i >= n - new:
            want.append(case["prompt"])
        elif r.random() < case["done"]:
            want.append(0)
        else:
            want.append(c + case["add"])
    return cached, want


def _node_counts(case):
    return _lens("nodes", case["seqs"], case["nodes"], 1) if case["ragged"] else [case["nodes"]] * case["seqs"]


def _trees(counts, words, r):
    """Ancestor masks (bit k of a row: it sees node k) of random trees in the order of their nodes, each node its own ancestor."""
    rows = []
    for t in counts:
        seen = []
        for i in range(t):
            parent = r.randint(max(-1, i - 6), i - 1) if i else -1
            seen.append((seen[parent] if parent >= 0 else 0) | (1 << i))
        rows += seen
    full = (1 << 64) - 1
    flat = [((m >> (64 * w)) & full) for m in rows for w in range(words)]
    flat = [x - (1 << 64) if x >> 63 else x for x in flat]
    return torch.tensor(flat, dtype=torch.int64).view(len(rows), words)


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


def _prepare_inputs(case, seed):
    cached, want = _row_lens(case)
    r = random.Random(seed)
    bs, n = case["block"], case["rows"]
    width = max(1, max(-(-max(c, w) // bs) for c, w in zip(cached, want)))
    held = sum(-(-c // bs) for c in cached)
    needed = sum(max(0, -(-w // bs) - -(-c // bs)) for c, w in zip(cached, want))
    blocks = held + needed + 64
    order = list(range(blocks))
    r.shuffle(order)
    rows = []
    for c in cached:
        own_blocks = [order.pop() for _ in range(-(-c // bs))]
        rows.append(own_blocks + [-1] * (width - len(own_blocks)))
    num_free = len(order)
    free = order + [-1] * (blocks - num_free)
    tokens = sum(max(0, w - c) for c, w in zip(cached, want))
    mask = None
    if case["tree"]:
        counts = [max(0, w - c) for c, w in zip(cached, want)]
        mask = _trees(counts, 1, r).cuda()
    return State(kind="inputs", tables=_int32(rows), cached=_int32(cached), want=_int32(want), free=_int32(free), num_free=_int32([num_free]), block=bs,
                 slots=blocks * bs, tokens=max(1, tokens + (tokens + 7) // 8 if not case["tree"] else tokens), mask=mask)


def _prepare_tree(case, seed):
    contexts = _lens("contexts", case["seqs"], case["longest"], case["shortest"])
    counts = _node_counts(case)
    r = random.Random(seed)
    bs, nkv, hd = case["block"], case["nkv"], case["hd"]
    lens = [c + t for c, t in zip(contexts, counts)]
    width = max(-(-c // bs) for c in lens)
    blocks = sum(-(-c // bs) for c in lens) + 3
    order = list(range(blocks))
    r.shuffle(order)
    rows = []
    for c in lens:
        mine = [order.pop() for _ in range(-(-c // bs))]
        rows.append(mine + [-1] * (width - len(mine)))
    g = _gpu(seed)
    k = torch.empty(blocks, bs, nkv, hd, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    v = torch.empty(blocks, bs, nkv, hd, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    q = torch.empty(sum(counts), case["nq"], hd, dtype=torch.bfloat16, device="cuda").normal_(0, 1.5, generator=g)
    words = -(-max(counts) // 64)
    return State(kind="tree", q=q, k=k, v=v, cu_q=_int32(_cumulative(counts)), lens=_int32(lens), tables=_int32(rows), mask=_trees(counts, words, r).cuda(),
                 max_q=max(counts), scale=hd ** -0.5, host_lens=lens, host_counts=counts, block=bs)


def _prepare_logits(case, seed):
    s, v, t = case["seqs"], case["vocab"], case["nodes"]
    rows = s * max(1, t)
    g, r = _gpu(seed), random.Random(seed)
    dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    logits = torch.empty(rows, v, dtype=dtype, device="cuda").normal_(0, 3, generator=g)
    st = State(kind="logits", logits=logits, vocab=v, args={})
    a = st.args
    if case["penalties"]:
        h = case["history"]
        lens = _lens("history", s, h, max(1, h // 2))
        # text repeats itself: the token ids crowd at the low end
        u = torch.empty(s, h, dtype=torch.float32, device="cuda").uniform_(generator=g)
        a["history"] = (u.pow_(4) * v).long().clamp_(0, v - 1)
        a["history_lens"] = _int32(lens)
        a["prompt_lens"] = _int32([r.randint(0, n) for n in lens])
        a["repetition_penalty"] = torch.tensor([r.choice((1.0, 1.05, 1.1, 1.3)) for _ in range(s)], device="cuda")
        a["presence_penalty"] = torch.tensor([r.choice((0.0, 0.5, 1.5)) for _ in range(s)], device="cuda")
        a["frequency_penalty"] = torch.tensor([r.choice((0.0, 0.1, 0.3)) for _ in range(s)], device="cuda")
    if case["bias"]:
        ids = torch.empty(s, case["bias"], dtype=torch.float32, device="cuda").uniform_(generator=g)
        ids = (ids * v).long().clamp_(0, v - 1)
        ids[:, case["bias"] - case["bias"] // 4:] = -1  # requests with fewer biases than the widest
        a["bias_ids"] = ids
        a["bias_values"] = torch.empty(s, case["bias"], device="cuda").uniform_(-5, 5, generator=g)
    if case["mask"]:
        bits = torch.randint(-2 ** 31, 2 ** 31, (rows, -(-v // 32)), dtype=torch.int64, device="cuda", generator=g).to(torch.int32)
        bits[::3] = -1  # rows without a grammar
        a["allowed_mask"] = bits
    if t:
        counts = [t] * s
        a["cu_seqlens"] = _int32(_cumulative(counts))
        a["draft_tokens"] = (torch.empty(rows, dtype=torch.float32, device="cuda").uniform_(generator=g).pow_(4) * v).long().clamp_(0, v - 1)
        a["tree_mask"] = _trees(counts, -(-t // 64), r).cuda()
    return st


def _package():
    import __graft_entry__
    package = __graft_entry__.load_package()
    from nanovllm_b200 import ops, runtime
    if runtime._RUNTIME is None:
        package.init_runtime(max_tokens=16384, hidden=4096)
    return ops


def prepare(case, seed):
    state = {"inputs": _prepare_inputs, "tree": _prepare_tree, "logits": _prepare_logits}[case["kind"]](case, seed)
    if own:
        state.ops = _package()
    return state


# ---- the plain forms -----------------------------------------------------------------------------------------------
def _popcount(words):
    """Set bits of the int64 words of each row."""
    bits = (words.unsqueeze(-1) >> torch.arange(64, device=words.device)) & 1
    return bits.sum((-1, -2))


def _visible(mask, nodes):
    """[rows, nodes] truth values of the ancestor masks."""
    k = torch.arange(nodes, device=mask.device)
    return ((mask[:, k // 64] >> (k % 64)) & 1).bool()


def _plain_inputs(s):
    tables, bs, (n, width) = s.tables, s.block, s.tables.shape
    c, t, dev = s.cached.long(), s.want.long(), s.tables.device
    full = width * bs
    valid = (c >= 0) & (c <= full) & (t >= 0) & (t <= full)
    c, t = c * valid, t * valid
    have, want = (c + bs - 1) // bs, (t + bs - 1) // bs
    add, need, back = (t - c).clamp(min=0), (want - have).clamp(min=0), (have - want).clamp(min=0)
    free = s.num_free.long().clamp(0, s.free.numel())
    top = free + back.sum()
    fits = add.cumsum(0) <= s.tokens
    granted = fits & ((need == 0) | (need.cumsum(0) <= top))  # the others stay as they are
    add, need = add * fits, need * granted
    lens = torch.where((t < c) | granted, t, c)
    zero = torch.zeros(1, dtype=torch.long, device=dev)
    cu_q, cu_k = torch.cat([zero, add.cumsum(0)]), torch.cat([zero, lens.cumsum(0)])
    # the stack with what came back on top of it
    back_end = back.cumsum(0)
    k = torch.arange(n * width, device=dev)
    row = torch.searchsorted(back_end, k, right=True).clamp(max=n - 1)
    col = (want[row] + k - (back_end - back)[row]).clamp(0, width - 1)
    returned = tables[row, col]
    # blocks taken from the top, in the order of the rows
    first = need.cumsum(0) - need
    j = torch.arange(width, device=dev) - have.unsqueeze(1)
    new = (j >= 0) & (j < need.unsqueeze(1))
    at = (top - 1 - (first.unsqueeze(1) + j)).clamp(min=0)
    block = torch.where(at < free, s.free[at.clamp(max=s.free.numel() - 1)], returned[(at - free).clamp(0, n * width - 1)])
    tables.copy_(torch.where(new, block, tables))
    left = (top - need.sum()).clamp(max=s.free.numel())
    i = torch.arange(s.free.numel(), device=dev)
    s.free.copy_(torch.where((i >= free) & (i < left), returned[(i - free).clamp(0, n * width - 1)], s.free))
    token = torch.arange(s.tokens, device=dev)
    row = torch.searchsorted(cu_q[1:], token, right=True)
    real = row < n
    row = row.clamp(max=n - 1)
    place = c[row] + token - cu_q[row]
    block = tables[row, (place // bs).clamp(0, width - 1)].long()
    slot = block * bs + place % bs
    slots = torch.where(real & granted[row] & (block >= 0) & (slot < s.slots), slot, -1)
    positions = place if s.mask is None else c[row] + (_popcount(s.mask) - 1).clamp(min=0)
    positions = torch.where(real, positions, 0)
    return (tables, s.free, positions, slots.int(), cu_q.int(), cu_k.int(), (cu_q[1:] - 1).clamp(min=0).int(), lens.int(), left.int())


def _plain_tree(s):
    nkv, hd = s.k.shape[2:]
    group = s.q.shape[1] // nkv
    outs, at = [], 0
    for i, (n, t) in enumerate(zip(s.host_lens, s.host_counts)):
        blocks = s.tables[i, :-(-n // s.block)].long()
        k = s.k[blocks].reshape(-1, nkv, hd)[:n].float().permute(1, 2, 0)
        v = s.v[blocks].reshape(-1, nkv, hd)[:n].float().transpose(0, 1)
        q = s.q[at:at + t].float().view(t, nkv, group, hd).permute(1, 2, 0, 3).reshape(nkv, group * t, hd)
        scores = (q @ k).view(nkv, group, t, n) * s.scale
        scores[..., n - t:].masked_fill_(~_visible(s.mask[at:at + t], t), float("-inf"))
        p = torch.exp(scores - scores.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        o = (p.view(nkv, group * t, n) @ v).view(nkv, group, t, hd)
        outs.append(o.permute(2, 0, 1, 3).reshape(t, nkv * group, hd).to(torch.bfloat16))
        at += t
    return torch.cat(outs)


def _plain_logits(s):
    a, (rows, v) = s.args, s.logits.shape
    x, dev = s.logits.float(), s.logits.device
    if "cu_seqlens" in a:
        row_seq = torch.searchsorted(a["cu_seqlens"][1:].long(), torch.arange(rows, device=dev), right=True)
    else:
        row_seq = torch.arange(rows, device=dev)
    if "history" in a:
        history, place = a["history"], torch.arange(a["history"].shape[1], device=dev)
        n, h = history.shape
        there = place < a["history_lens"].unsqueeze(1)
        output = there & (place >= a["prompt_lens"].unsqueeze(1))
        counts = torch.zeros(n, v, device=dev).scatter_add_(1, history, output.float())[row_seq]
        seen = torch.zeros(n, v, device=dev).scatter_add_(1, history, there.float())[row_seq]
        if "draft_tokens" in a:
            first = a["cu_seqlens"].long()[row_seq]
            for k in range(64 * a["tree_mask"].shape[1]):
                node = (first + k).clamp(max=rows - 1)
                sees = ((a["tree_mask"][:, k // 64] >> (k % 64)) & 1).bool() & (first + k < a["cu_seqlens"].long()[row_seq + 1])
                counts.scatter_add_(1, a["draft_tokens"][node].unsqueeze(1), sees.float().unsqueeze(1))
                seen.scatter_add_(1, a["draft_tokens"][node].unsqueeze(1), sees.float().unsqueeze(1))
        r = a["repetition_penalty"][row_seq].unsqueeze(1)
        x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
        x = x - a["frequency_penalty"][row_seq].unsqueeze(1) * counts
        x = x - a["presence_penalty"][row_seq].unsqueeze(1) * (counts > 0)
    if "bias_ids" in a:
        ids, values = a["bias_ids"], a["bias_values"]
        later = torch.arange(ids.shape[1], device=dev)
        shadowed = ((ids.unsqueeze(1) == ids.unsqueeze(2)) & (later.unsqueeze(0) > later.unsqueeze(1))).any(-1)  # the last of equal ids counts
        bias = torch.zeros(ids.shape[0], v, device=dev).scatter_add_(1, ids.clamp(min=0), torch.where(shadowed | (ids < 0), 0.0, values))
        x = x + bias[row_seq]
    if "allowed_mask" in a:
        token = torch.arange(v, device=dev)
        x = torch.where(((a["allowed_mask"][:, token // 32] >> (token % 32)) & 1).bool(), x, float("-inf"))
    return x.to(s.logits.dtype)


# ---- the calls -----------------------------------------------------------------------------------------------------
def run(state):
    s = state
    if not own:
        return {"inputs": _plain_inputs, "tree": _plain_tree, "logits": _plain_logits}[s.kind](s)
    if s.kind == "inputs":
        return (s.tables, s.free, *s.ops.batch_inputs(s.tables, s.cached, s.want, s.free, s.num_free, s.block, s.slots, s.tokens, tree_mask=s.mask))
    if s.kind == "tree":
        return s.ops.tree_attention(s.q, s.k, s.v, s.cu_q, s.lens, s.tables, s.mask, s.max_q, s.scale)
    return s.ops.adjust_logits(s.logits, **s.args)


# ---- what a pass cannot do without -------------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "inputs":
        cached, want = _row_lens(case)
        bs, n = case["block"], case["rows"]
        tokens = sum(max(0, w - c) for c, w in zip(cached, want))
        moved = sum(abs(-(-w // bs) - -(-c // bs)) for c, w in zip(cached, want))  # blocks taken and given back
        touched = sum(1 for c, w in zip(cached, want) if w > c and c % bs)  # open blocks, whose numbers are read
        return {"bytes": 12 * tokens + (8 * tokens if case["tree"] else 0) + 8 * n + 16 * n + 8 * moved + 4 * touched + 16, "flops": 4 * tokens + 8 * n}
    if case["kind"] == "tree":
        contexts = _lens("contexts", case["seqs"], case["longest"], case["shortest"])
        counts = _node_counts(case)
        keys = sum(contexts) + sum(counts)
        pairs = sum(t * (c + t) for c, t in zip(contexts, counts))
        return {"bytes": 4 * keys * case["nkv"] * case["hd"] + 4 * sum(counts) * case["nq"] * case["hd"] + 8 * sum(counts) * -(-max(counts) // 64) + 4 * keys // case["block"],
                "flops": 4 * pairs * case["nq"] * case["hd"]}
    s, v, t = case["seqs"], case["vocab"], case["nodes"]
    rows, size = s * max(1, t), 2 if case["dtype"] == "bf16" else 4
    moved = 2 * size * rows * v
    if case["penalties"]:
        moved += 8 * sum(_lens("history", s, case["history"], max(1, case["history"] // 2))) + 20 * s
    if case["mask"]:
        moved += 4 * rows * -(-v // 32)
    return {"bytes": moved + 12 * s * case["bias"] + (16 * rows if t else 0), "flops": rows * v}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
def _exact_inputs(s):
    """A request at a time, as a block manager on the host does it."""
    tables, free = s.tables.tolist(), s.free.tolist()
    cached, want, bs, width = s.cached.tolist(), s.want.tolist(), s.block, s.tables.shape[1]
    top = min(max(0, s.num_free.item()), len(free))
    stack, depths = free[:top], None if s.mask is None else [bin(w & (1 << 64) - 1).count("1") for w in s.mask[:, 0].tolist()]
    for i, (c, t) in enumerate(zip(cached, want)):
        stack += [tables[i][j] for j in range(-(-t // bs), -(-c // bs))]
    positions, slots, cu_q, cu_k, lens = [], [], [0], [0], []
    for i, (c, t) in enumerate(zip(cached, want)):
        for j in range(-(-c // bs), -(-t // bs)):
            tables[i][j] = stack.pop()
        for p in range(c, t):
            positions.append(p if depths is None else c + depths[len(positions)] - 1)
            slots.append(tables[i][p // bs] * bs + p % bs)
        lens.append(t)
        cu_q.append(len(slots))
        cu_k.append(cu_k[-1] + t)
    pad = s.tokens - len(slots)
    free[top:max(top, len(stack))] = stack[top:]
    return (_int32(tables), _int32(free), torch.tensor(positions + [0] * pad, device="cuda"), _int32(slots + [-1] * pad), _int32(cu_q), _int32(cu_k),
            _int32([max(0, x - 1) for x in cu_q[1:]]), _int32(lens), _int32([len(stack)]))


def _exact_tree(s):
    nq, hd = s.q.shape[1:]
    nkv = s.k.shape[2]
    out, at = torch.empty(s.q.shape, dtype=torch.float64, device="cuda"), 0
    for i, (n, t) in enumerate(zip(s.host_lens, s.host_counts)):
        place = torch.arange(n, device="cuda")
        slot = s.tables[i].long()[place // s.block] * s.block + place % s.block
        sees = torch.ones(t, n, dtype=torch.bool, device="cuda")
        for row, words in enumerate(s.mask[at:at + t].tolist()):
            sees[row, n - t:] = torch.tensor([bool(words[k // 64] >> (k % 64) & 1) for k in range(t)])
        for h in range(nkv):
            keys, values = s.k.view(-1, nkv, hd)[slot, h].double(), s.v.view(-1, nkv, hd)[slot, h].double()
            for q in range(h * nq // nkv, (h + 1) * nq // nkv):
                score = torch.where(sees, s.q[at:at + t, q].double() @ keys.T * s.scale, float("-inf"))
                out[at:at + t, q] = torch.softmax(score, -1) @ values
        at += t
    return out


def _exact_logits(s):
    a, (rows, v) = s.args, s.logits.shape
    cu = a["cu_seqlens"].tolist() if "cu_seqlens" in a else list(range(rows + 1))
    out = torch.empty(rows, v, dtype=torch.float64, device="cuda")
    for i, (first, last) in enumerate(zip(cu[:-1], cu[1:])):
        bias = {}
        if "bias_ids" in a:
            bias = {k: b for k, b in zip(a["bias_ids"][i].tolist(), a["bias_values"][i].tolist()) if k >= 0}
        if "history" in a:
            text = a["history"][i, :a["history_lens"][i]]
            prompt, said = text[:a["prompt_lens"][i]], text[a["prompt_lens"][i]:]
        for row in range(first, last):
            x = s.logits[row].double()
            if "history" in a:
                mine = said
                if "draft_tokens" in a:
                    words = a["tree_mask"][row].tolist()
                    path = [k for k in range(last - first) if words[k // 64] >> (k % 64) & 1]
                    mine = torch.cat([said, a["draft_tokens"][[first + k for k in path]]])
                times = torch.bincount(mine, minlength=v).double()
                known = (times + torch.bincount(prompt, minlength=v)) > 0
                factor = a["repetition_penalty"][i].double()
                x = x * torch.where(known, torch.where(x > 0, 1 / factor, factor), 1.0)
                x = x - a["frequency_penalty"][i].double() * times - a["presence_penalty"][i].double() * times.clamp(max=1)
            if bias:
                x[list(bias)] += torch.tensor(list(bias.values()), dtype=torch.float64, device="cuda")
            if "allowed_mask" in a:
                bits = (a["allowed_mask"][row].unsqueeze(1) >> torch.arange(32, device="cuda")) & 1
                x[bits.view(-1)[:v] == 0] = float("-inf")
            out[row] = x
    return out


def exact(case, seed):
    state = {"inputs": _prepare_inputs, "tree": _prepare_tree, "logits": _prepare_logits}[case["kind"]](case, seed)
    return {"inputs": _exact_inputs, "tree": _exact_tree, "logits": _exact_logits}[case["kind"]](state)
