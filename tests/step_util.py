"""Plain statements of a verification step's operators, for their tests: whole numbers on the host, the rest in 64 bits."""
import random

import torch


def trees(counts, words, seed, reach=6):
    """Ancestor masks (int64 [sum(counts), words]) and parents of random trees; every node sees itself."""
    r = random.Random(seed)
    rows = []
    for t in counts:
        seen = []
        for i in range(t):
            parent = r.randint(max(-1, i - reach), i - 1) if i else -1
            seen.append((seen[parent] if parent >= 0 else 0) | (1 << i))
        rows += seen
    return masks(rows, words)


def masks(rows, words):
    """Whole numbers of any size as rows of int64 words."""
    flat = [(m >> (64 * w)) & ((1 << 64) - 1) for m in rows for w in range(words)]
    return torch.tensor([x - (1 << 64) if x >> 63 else x for x in flat], dtype=torch.int64).view(len(rows), words)


def bits(mask, n):
    """[rows, n] truth values of the first n bits (zero past the words)."""
    k = torch.arange(n)
    words = torch.cat([mask.cpu(), torch.zeros(mask.shape[0], -(-n // 64) + 1, dtype=torch.int64)], 1)
    return ((words[:, k // 64] >> (k % 64)) & 1).bool()


def cumulative(counts):
    return torch.tensor([0] + list(counts)).cumsum(0).to(torch.int32)


def batch_inputs(tables, cached, wanted, free, num_free, bs, num_slots, max_tokens, mask=None):
    """The requests one after the other, on lists.  Returns tables, free, then the results in their order."""
    tables, free, width = [list(t) for t in tables], list(free), len(tables[0]) if tables else 0
    full = width * bs

    def blocks(x):
        return -(-x // bs)

    pairs = [(c, w) if 0 <= c <= full and 0 <= w <= full else (0, 0) for c, w in zip(cached, wanted)]
    top = min(max(0, num_free), len(free))
    stack = free[:top]
    for i, (c, w) in enumerate(pairs):
        stack += tables[i][blocks(w):blocks(c)]
    room, asked_tokens, asked_blocks = len(stack), 0, 0
    positions, slots, cu_q, cu_k, last, lens = [], [], [0], [0], [], []
    for i, (c, w) in enumerate(pairs):
        add, need = max(0, w - c), max(0, blocks(w) - blocks(c))
        asked_tokens += add
        asked_blocks += need
        fits = asked_tokens <= max_tokens
        granted = fits and (need == 0 or asked_blocks <= room)
        if granted:
            for j in range(need):
                tables[i][blocks(c) + j] = stack.pop()
        for p in range(c, w) if fits else ():
            at = len(positions)
            positions.append(p if mask is None else c + max(0, int(bits(mask[at:at + 1], min(add, 64 * mask.shape[1])).sum()) - 1))
            slot = tables[i][p // bs] * bs + p % bs if granted else -1
            slots.append(slot if granted and tables[i][p // bs] >= 0 and slot < num_slots else -1)
        lens.append(w if w < c or granted else c)
        cu_q.append(len(slots))
        cu_k.append(cu_k[-1] + lens[-1])
        last.append(max(0, len(slots) - 1))
    left = min(len(stack), len(free))
    free[top:max(top, left)] = stack[top:max(top, left)]
    pad = max_tokens - len(slots)
    return tables, free, positions + [0] * pad, slots + [-1] * pad, cu_q, cu_k, last, lens, [left]


def tree_attention(q, k_cache, v_cache, counts, lens, tables, mask, scale):
    """The definition in 64 bits, and the sum of |p v| that bounds what rounding the probabilities does."""
    nq, hd = q.shape[1:]
    bs, nkv = k_cache.shape[1:3]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    at = 0
    for b, (t, n) in enumerate(zip(counts, lens)):
        if n >= t > 0 and n > 0:
            place = torch.arange(n, device=q.device)
            slot = tables[b].long()[place // bs] * bs + place % bs
            sees = torch.ones(t, n, dtype=torch.bool, device=q.device)
            sees[:, n - t:] = bits(mask[at:at + t], t).to(q.device)
            for h in range(nkv):
                k, v = k_cache.view(-1, nkv, hd)[slot, h].double(), v_cache.view(-1, nkv, hd)[slot, h].double()
                group = nq // nkv
                x = q[at:at + t, h * group:(h + 1) * group].double()
                s = torch.einsum("tgd,nd->tgn", x, k) * scale
                s = torch.where(sees.unsqueeze(1), s, float("-inf"))
                p = torch.where(sees.unsqueeze(1), torch.exp(s - s.amax(-1, keepdim=True)), 0.0)
                total = p.sum(-1, keepdim=True)
                p = torch.where(total > 0, p / total, 0.0)
                # (a node that is not seen may hold anything: its values are left out, not multiplied by zero)
                live = sees.any(0)
                if torch.isfinite(v[live]).all():
                    v = torch.where(live.unsqueeze(1), v, 0.0)
                    out[at:at + t, h * group:(h + 1) * group] = torch.einsum("tgn,nd->tgd", p, v)
                    size[at:at + t, h * group:(h + 1) * group] = torch.einsum("tgn,nd->tgd", p, v.abs())
                else:
                    for i in range(t):
                        out[at + i, h * group:(h + 1) * group] = p[i][:, sees[i]] @ v[sees[i]]
                        size[at + i, h * group:(h + 1) * group] = p[i][:, sees[i]] @ v[sees[i]].abs()
        at += t
    return out, size


def adjust_logits(logits, history=None, history_lens=None, prompt_lens=None, repetition_penalty=None, presence_penalty=None, frequency_penalty=None,
                  bias_ids=None, bias_values=None, allowed_mask=None, cu_seqlens=None, draft_tokens=None, tree_mask=None):
    """A row at a time in 64 bits; everything on the CPU."""
    rows, vocab = logits.shape
    cu = list(range(rows + 1)) if cu_seqlens is None else cu_seqlens.tolist()
    out = logits.double().clone()
    for s in range(len(cu) - 1):
        prompt, said = [], []
        if history is not None:
            n = max(0, min(int(history_lens[s]), history.shape[1]))
            p = 0 if prompt_lens is None else max(0, min(int(prompt_lens[s]), n))
            prompt, said = history[s, :p].tolist(), history[s, p:n].tolist()
        bias = {}
        if bias_ids is not None:
            bias = {t: b for t, b in zip(bias_ids[s].tolist(), bias_values[s].double().tolist()) if 0 <= t < vocab}
        for row in range(cu[s], min(rows, cu[s + 1])):
            x, path = out[row], []
            if draft_tokens is not None:
                path = [int(draft_tokens[cu[s] + k]) for k in range(cu[s + 1] - cu[s]) if k < 64 * tree_mask.shape[1] and bool(bits(tree_mask[row:row + 1], k + 1)[0, k])]
            count = {}
            for t in said + path:
                if 0 <= t < vocab:
                    count[t] = count.get(t, 0) + 1
            for t in {t for t in prompt if 0 <= t < vocab} | set(count):
                if repetition_penalty is not None:
                    x[t] = x[t] / repetition_penalty[s].double() if x[t] > 0 else x[t] * repetition_penalty[s].double()
                if t in count:
                    x[t] -= (0 if frequency_penalty is None else frequency_penalty[s].double() * count[t]) + (0 if presence_penalty is None else presence_penalty[s].double())
            for t, b in bias.items():
                x[t] += b
            if allowed_mask is not None:
                words = allowed_mask[row].long() & 0xffffffff
                k = torch.arange(vocab)
                x[((words[k // 32] >> (k % 32)) & 1) == 0] = float("-inf")
    return out
