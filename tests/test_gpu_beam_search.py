"""A beam search on one B200: the operators of its steps together, on a model of one table, and ModelRunner.beam_search on a small random-init Qwen3."""
import pytest
import torch

import beam_util as ref
from tests.gpu_util import ensure_group
from tests.test_gpu_model import _attention_backend

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def runner(pkg):
    ensure_group()
    from nanovllm_b200.engine.model_runner import ModelConfig, ModelRunner
    _attention_backend()
    cfg = ModelConfig(hidden_size=1024, num_attention_heads=8, num_key_value_heads=4, head_dim=128, intermediate_size=2048, num_hidden_layers=3, vocab_size=2048,
                      max_position_embeddings=2048)
    runner = ModelRunner(cfg, max_num_seqs=64, max_model_len=1024, max_num_batched_tokens=2048, kvcache_block_size=16, num_kvcache_blocks=400, enforce_eager=True, oneshot_tokens=128, seed=3)
    yield runner
    runner.exit()


def sequences(lens, seed, first=0):
    from nanovllm_b200.engine.model_runner import Seq
    g = torch.Generator().manual_seed(seed)
    out, at = [], first
    for n in lens:
        blocks = -(-n // 16)
        out.append(Seq(torch.randint(0, 2048, (n,), generator=g).tolist(), list(range(at, at + blocks))))
        at += blocks
    return out


def logits_after(runner, prompt, token_lists):
    """The model's logits after the prompt and each of the lists of tokens, from one prefill a list (float64, on the host)."""
    from nanovllm_b200.engine.model_runner import Seq
    from nanovllm_b200.utils.context import reset_context
    blocks = -(-(len(prompt) + max(map(len, token_lists))) // 16)
    seqs = [Seq(prompt + t, list(range(200 + i * blocks, 200 + (i + 1) * blocks))) for i, t in enumerate(token_lists)]
    assert 200 + len(seqs) * blocks <= 400
    ids, pos = runner.prepare_prefill(seqs)
    out = runner.run_model(ids, pos, True).double().cpu()
    reset_context()
    return out


# A logit is off by two roundings to bf16 of its size between the paths (2^-8 each, sizes up to 4 here), the log of the sum by as much: 0.0625 a token.
STEP = 0.0625


@pytest.mark.parametrize("lens, beams, new", [([20], 4, 6), ([37, 16, 1], 3, 20), ([100, 33], 8, 5), ([15], 1, 4), ([48], 32, 3)])
def test_sums_are_the_models(runner, lens, beams, new):
    """Every continuation's sum is that of the log-probabilities that the model gives its tokens in one prefill, and the first is no worse than decoding the best token each time.  That is
    so only where tables, copies and histories follow the beams: a block of another beam changes every later logit."""
    seqs = sequences(lens, seed=len(lens) + beams)
    found = runner.beam_search(seqs, beams, new, list(range(100, 399)))
    assert [len(f) for f in found] == [beams] * len(lens)
    for s, continuations in zip(seqs, found):
        assert len({tuple(t) for t, _ in continuations}) == beams and all(len(t) == new for t, _ in continuations)
        scores = [x for _, x in continuations]
        assert scores == sorted(scores, reverse=True)
        prompt = list(s.token_ids)
        for tokens, score in (continuations if beams <= 8 else continuations[:2] + continuations[-2:]):
            rows = torch.cat([logits_after(runner, prompt, [tokens[:i]]) for i in range(new)])
            want = rows.log_softmax(-1).gather(1, torch.tensor(tokens)[:, None]).sum().item()
            assert abs(want - score) <= STEP * new, (want, score)
        greedy, total = [], 0.0
        for _ in range(new):
            row = logits_after(runner, prompt, [greedy])[0].log_softmax(-1)
            greedy.append(row.argmax().item())
            total += row.max().item()
        if beams == 1:
            assert abs(total - scores[0]) <= 2 * STEP * new  # (a step may pick another token as good)


def test_the_first_step_is_the_best_tokens(runner):
    seqs = sequences([30, 5], seed=9)
    found = runner.beam_search(seqs, 6, 1, list(range(100, 200)))
    for s, f in zip(seqs, found):
        row = logits_after(runner, list(s.token_ids), [[]])[0].log_softmax(-1)
        for tokens, score in f:
            assert abs(row[tokens[0]].item() - score) <= STEP
        assert min(x for _, x in f) >= row.topk(6).values[-1].item() - 2 * STEP


def test_ends_and_rules(runner):
    """A beam ends with eos_token and keeps its sum; a rule that leaves two tokens leaves their continuations only, fewer than there are beams."""
    seqs = sequences([20, 40], seed=11)
    allowed = torch.zeros(2, 64, dtype=torch.int32, device=DEV)
    allowed[:, 0] = 0b110  # tokens 1 and 2
    found = runner.beam_search(seqs, 8, 2, list(range(100, 200)), rules=dict(allowed_mask=allowed))
    assert all(sorted(t for t, _ in f) == [[1, 1], [1, 2], [2, 1], [2, 2]] for f in found)
    found = runner.beam_search(seqs, 8, 3, list(range(100, 200)), rules=dict(allowed_mask=allowed), eos_token=2)
    assert all(sorted(t for t, _ in f) == [[1, 1, 1], [1, 1, 2], [1, 2], [2]] for f in found)
    found = runner.beam_search(seqs, 8, 30, list(range(100, 200)), rules=dict(allowed_mask=allowed & 0b100), eos_token=2)
    assert all([t for t, _ in f] == [[2]] for f in found)  # (all have ended after one step)
    # histories: tokens that have occurred, in the prompt or in the beam, are pushed away
    plain = runner.beam_search(seqs, 4, 6, list(range(100, 200)))
    fresh = runner.beam_search(seqs, 4, 6, list(range(100, 200)), rules=dict(presence_penalty=torch.full((2,), 100.0, device=DEV)))
    assert all(len(set(t)) == len(t) for f in fresh for t, _ in f)
    assert runner.beam_search(seqs, 4, 6, list(range(100, 200))) == plain


def test_refusals(runner):
    from nanovllm_b200.utils.context import get_context
    seqs = sequences([20], seed=13)
    free = list(range(100, 200))
    assert runner.beam_search([], 4, 5, free) == []
    for args in ((seqs, 0, 5, free), (seqs, 33, 5, free), (seqs, 4, 0, free), (seqs * 20, 4, 5, free), (seqs, 4, 2000, free), (seqs, 4, 30, free[:3]), (sequences([20, 0], 1), 4, 5, free)):
        with pytest.raises(ValueError):
            runner.beam_search(*args)
    for blocks in ([100] * 50, list(range(50)), list(range(380, 430)), [-1] + free):
        with pytest.raises(ValueError, match="blocks"):
            runner.beam_search(seqs, 4, 5, blocks)
    shared = sequences([20, 20], seed=13)
    shared[1].block_table = list(shared[0].block_table)
    with pytest.raises(ValueError, match="share"):
        runner.beam_search(shared, 4, 5, free)
    seqs[0].block_table = [0]
    with pytest.raises(ValueError, match="room"):
        runner.beam_search(seqs, 4, 5, free)
    seqs = sequences([20], seed=13)
    seqs[0].num_cached_tokens = 20
    with pytest.raises(ValueError):
        runner.beam_search(seqs, 4, 5, free)
    seqs[0].num_cached_tokens = 0
    with pytest.raises(ValueError):
        runner.beam_search(seqs, 4, 5, free, rules=dict(bias_ids=torch.zeros(2, 1, dtype=torch.int64, device=DEV), bias_values=torch.zeros(1, 1, device=DEV)))
    assert get_context().prefix_lens is None
    assert len(runner.beam_search(seqs, 2, 2, free)[0]) == 2


@pytest.mark.parametrize("graphed", [False, True])
def test_a_search_by_hand(runner, graphed):
    """The operators in a serving program's loop, eager and as one captured step that is replayed, against the same search on the host.  The keys of a token are its own row of a table, so that
    the model is: attention over the beam's tokens, and logits from its result.  In every step the new beams are continuations of the ones before with their sums, and none that
    was left out is better by more than the bf16 attention results allow: a result of size about 1 is off by 2^-7 at most, a logit is 128 of them with weights of 0.3, whose errors add up like
    their squares, 0.3 * sqrt(128) * 2^-8 (two standard deviations: 0.03), and so is the log of the sum: 0.05."""
    from nanovllm_b200 import ops
    n, beams, vocab, bs, nkv, nq, hd, steps, prompt_len = 3, 4, 500, 16, 1, 2, 64, 20, 37
    g = torch.Generator(device=DEV).manual_seed(1)
    table_k, table_v, table_q = (torch.randn(vocab, heads, hd, device=DEV, generator=g).bfloat16() for heads in (nkv, nkv, nq))
    out_w = (torch.randn(nq * hd, vocab, device=DEV, generator=g) * 0.3)
    prompts = torch.randint(0, vocab, (n, prompt_len), generator=torch.Generator().manual_seed(2))
    rows, width, blocks, full = n * beams, 5, 64, prompt_len // bs
    cache = torch.full((2, 1, blocks, bs, nkv, hd), float("nan"), dtype=torch.bfloat16, device=DEV)
    tables = torch.full((rows, width), -1, dtype=torch.int32)
    for r in range(n):
        tables[r * beams, :3] = torch.tensor([3 * r, 3 * r + 1, 3 * r + 2])
        for i in range(prompt_len - 1):  # (the last token goes in with the first step)
            cache[0, 0, 3 * r + i // bs, i % bs], cache[1, 0, 3 * r + i // bs, i % bs] = table_k[prompts[r, i]], table_v[prompts[r, i]]
    live = torch.arange(rows) % beams == 0
    st = dict(tables=tables.to(DEV), lens=torch.where(live, prompt_len - 1, 0).int().to(DEV), stack=torch.cat([torch.arange(9, blocks), torch.zeros(9)]).int().to(DEV),
              height=torch.tensor([blocks - 9], dtype=torch.int32, device=DEV), scores=torch.where(live, 0.0, float("-inf")).view(n, beams).to(DEV),
              tokens=prompts[:, -1:].repeat(1, beams).contiguous().to(DEV), ended=torch.zeros(n, beams, dtype=torch.bool, device=DEV),
              history=torch.zeros(rows, steps, dtype=torch.int64, device=DEV), said=torch.zeros(rows, dtype=torch.int32, device=DEV))
    cu, prefix, first = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (range(0, rows + 1, beams), [full * bs] * n, [full] * n))

    def step():
        inputs = ops.batch_inputs(st["tables"], st["lens"], st["lens"] + 1, st["stack"], st["height"], bs, blocks * bs, rows)
        ids = st["tokens"].view(rows).clamp(min=0)
        ops.store_kvcache(table_k[ids], table_v[ids], cache[0, 0], cache[1, 0], inputs.slot_mapping)
        seen = torch.where(st["ended"].view(rows) | (st["lens"] == 0), 0, inputs.context_lens)
        o = ops.shared_prefix_attention(table_q[ids], cache[0, 0], cache[1, 0], cu, prefix, seen, st["tables"], beams, hd ** -0.5)
        picks = ops.beam_select(o.view(rows, -1).float() @ out_w, st["scores"], beams, finished=st["ended"], eos_token=7)
        state = ops.reorder_beams(picks.parents, st["tables"], inputs.context_lens, st["stack"], inputs.num_free, cache, first_blocks=first, history=st["history"], history_lens=st["said"],
                                  tokens=picks.tokens)
        for name, x in (("tables", state.block_tables), ("lens", state.context_lens), ("height", state.num_free), ("scores", picks.scores), ("tokens", picks.tokens), ("ended", picks.finished),
                        ("history", state.history), ("said", state.history_lens)):
            st[name].copy_(x)

    # all continuations of a request's beams (tokens, sum, at its end), by the definition: (their tokens, sum, at its end)
    kh, vh, qh, wh = (x.double().cpu() for x in (table_k, table_v, table_q, out_w))

    def continuations(r, host):
        out = []
        for said, score, ended in host:
            if score == float("-inf"):
                continue
            if ended:
                out.append((said, score, True))
                continue
            seq = prompts[r].tolist() + said
            p = torch.softmax(hd ** -0.5 * torch.einsum("hd,kd->hk", qh[seq[-1]], kh[seq, 0]), -1)
            row = (torch.einsum("hk,kd->hd", p, vh[seq, 0]).reshape(-1) @ wh).log_softmax(-1).tolist()
            out += [(said + [t], score + x, t == 7) for t, x in enumerate(row)]
        return out

    graph = None
    if graphed:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        torch.matmul(torch.zeros(rows, nq * hd, device=DEV), out_w)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
    beams_of = [[([], 0.0, False)] for _ in range(n)]
    for _ in range(steps):
        graph.replay() if graphed else step()
        torch.cuda.synchronize()
        said, text, scores, ended = (st[x].tolist() for x in ("said", "history", "scores", "ended"))
        tables_now, lens = st["tables"].tolist(), st["lens"].tolist()
        for r in range(n):
            # the device's own bookkeeping: a row's cache holds its tokens' rows, whatever beams it came from
            for b in range(beams):
                row = r * beams + b
                seq = prompts[r].tolist() + text[row][:said[row]]
                count = min(lens[row], len(seq) - 1)  # (a beam at its end goes on growing)
                at = [tables_now[row][i // bs] * bs + i % bs for i in range(count)]
                assert torch.equal(cache[0, 0].view(-1, nkv, hd)[at], table_k[seq[:count]])
            now = [(text[r * beams + b][:said[r * beams + b]], scores[r][b], ended[r][b]) for b in range(beams)]
            want = {tuple(t): (x, e) for t, x, e in continuations(r, beams_of[r])}
            assert len({tuple(t) for t, _, _ in now}) == beams
            for t, x, e in now:
                assert abs(want[tuple(t)][0] - x) <= 0.05 and want[tuple(t)][1] == e
            picked = {tuple(t) for t, _, _ in now}
            assert max(x for t, (x, _) in want.items() if t not in picked) <= min(want[t][0] for t in picked) + 2 * 0.05
            beams_of[r] = now
    used = {b for row, l in zip(tables_now, lens) for b in row[:-(-l // bs)]}
    height = st["height"].item()
    left = set(st["stack"].tolist()[:height])
    assert len(left) == height and not left & used and len(left | used | set(range(3 * n))) == blocks, "blocks were lost or given twice"
