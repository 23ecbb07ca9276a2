"""Plain definitions of the operators of a beam-search step, in 64 bits and on the host, for the tests."""
import torch


def shared_prefix_attention(q, k_cache, v_cache, cu_groups, context_lens, block_tables, scale):
    """Each sequence's attention over its own table; (out, weighted mean of |v|), float64 [n, nq, hd].  Sequences without tokens or group: zeros."""
    n, nq, hd = q.shape
    bs, nkv = k_cache.shape[1], k_cache.shape[2]
    k_rows, v_rows = k_cache.reshape(-1, nkv, hd), v_cache.reshape(-1, nkv, hd)
    out, size = torch.zeros(n, nq, hd, dtype=torch.float64, device=q.device), torch.zeros(n, nq, hd, dtype=torch.float64, device=q.device)
    cu = [max(0, min(c, n)) for c in cu_groups]
    grouped = {s for a, b in zip(cu, cu[1:]) for s in range(a, b)}
    for s in range(n):
        length = context_lens[s]
        if length <= 0 or s not in grouped:
            continue
        at = torch.tensor([block_tables[s][i // bs] * bs + i % bs for i in range(length)], device=q.device)
        k, v = (rows[at].double().repeat_interleave(nq // nkv, dim=1) for rows in (k_rows, v_rows))
        p = torch.softmax(scale * torch.einsum("hd,khd->hk", q[s].double(), k), dim=-1)
        out[s], size[s] = torch.einsum("hk,khd->hd", p, v), torch.einsum("hk,khd->hd", p, v.abs())
    return out, size


def beam_select(logits, scores, picks, finished=None, eos_token=None):
    """(scores float64, parents, tokens, finished), [n, picks], as lists; logits [n * beams, vocab]."""
    n, beams = scores.shape
    vocab = logits.shape[1]
    x, s = logits.double().cpu(), scores.double().cpu()
    largest = torch.finfo(logits.dtype).max
    x = torch.where(x == float("inf"), largest, x)
    x = torch.where(x.isnan(), float("-inf"), x)
    out = ([], [], [], [])
    for r in range(n):
        rows, kinds = [], []
        for b in range(beams):
            row = torch.full((vocab,), float("-inf"), dtype=torch.float64)
            ended = finished is not None and bool(finished[r, b])
            if s[r, b] > float("-inf"):  # (not for NaN)
                if ended:
                    row[0] = s[r, b]
                elif (x[r * beams + b] > float("-inf")).any():
                    y = x[r * beams + b]
                    top = y.max()
                    row = s[r, b] + ((y - top) - (y - top).exp().sum().log())
            rows.append(row)
            kinds.append(ended)
        flat = torch.cat(rows)
        value, order = torch.sort(flat, descending=True, stable=True)  # of equal ones the lowest beam, then the lowest token
        best = [(value[i].item(), order[i].item()) for i in range(min(picks, flat.numel())) if value[i] > float("-inf")]
        pad = picks - len(best)
        out[0].append([v for v, _ in best] + [float("-inf")] * pad)
        out[1].append([o // vocab for _, o in best] + [-1] * pad)
        out[2].append([-1 if kinds[o // vocab] else o % vocab for _, o in best] + [-1] * pad)
        out[3].append([kinds[o // vocab] or (eos_token is not None and o % vocab == eos_token) for _, o in best] + [False] * pad)
    return out


def reorder_beams(parents, tables, lens, free, num_free, block_size, cache_blocks, first_blocks=None):
    """parents: lists per request.  (tables, lens, stack, its height, copies): copies are (from, to, tokens)."""
    beams, width = len(parents[0]) if parents else 1, len(tables[0]) if tables else 0
    stack, height = list(free), max(0, min(num_free, len(free)))
    new_tables, new_lens, given, wants = [], [], [], []

    def entry(row, column):
        b = tables[row][column]
        return b if 0 <= b < cache_blocks else -1

    for r, request in enumerate(parents):
        old = range(r * beams, (r + 1) * beams)
        length = [lens[o] if 0 <= lens[o] <= width * block_size else 0 for o in old]
        have = [-(-n // block_size) for n in length]
        taken = {}  # (column, block) that keeps its first row
        for b, p in enumerate(request):
            row = [-1] * width
            if not 0 <= p < beams:
                new_tables.append(row)
                new_lens.append(0)
                continue
            n = length[p]
            for c in range(have[p]):
                row[c] = entry(r * beams + p, c)
            if n % block_size:
                c = n // block_size
                if row[c] >= 0:
                    # the first row of the new ones that has this block in this column keeps it, whether it goes on in it or not
                    holders = [q for q in request[:b] if 0 <= q < beams and c < have[q] and entry(r * beams + q, c) == row[c]]
                    if holders:
                        wants.append((len(new_tables), c, row[c], n - c * block_size))
            new_tables.append(row)
            new_lens.append(n)
        first = first_blocks[r] if first_blocks is not None else 0
        kept = {(c, entry(r * beams + p, c)) for p in request if 0 <= p < beams for c in range(have[p])}
        seen = set()
        for c in range(width):
            for i, o in enumerate(old):
                if c >= have[i] or c < min(first, length[i] // block_size):
                    continue
                block = entry(o, c)
                if block >= 0 and (c, block) not in kept and (c, block) not in seen:
                    seen.add((c, block))
                    given.append(block)
    room, stack = len(stack), stack[:height] + given + stack[height + len(given):]  # (what does not fit after the copies have taken theirs is lost)
    height += len(given)
    copies = []
    for row, c, block, tokens in wants:
        to = -1
        if height > 0:
            height -= 1
            to = stack[height]
            if not 0 <= to < cache_blocks:
                to = -1
        if to < 0:
            new_tables[row][c], new_lens[row] = -1, c * block_size
        else:
            new_tables[row][c] = to
            copies.append((block, to, tokens))
    return new_tables, new_lens, stack[:room], min(height, room), copies


def append_history(parents, history, lens, tokens, width):
    beams = len(parents[0])
    out, said = [], []
    for r, request in enumerate(parents):
        for b, p in enumerate(request):
            if not 0 <= p < beams:
                row = []
            else:
                at = r * beams + p
                row = list(history[at][:max(0, min(lens[at], width))])
                if tokens is not None and tokens[r][b] >= 0 and len(row) < width:
                    row.append(tokens[r][b])
            out.append(row + [-1] * (width - len(row)))
            said.append(len(row))
    return out, said
