"""The part of the model runner that hosts the tensor-parallel layer path.

It covers what nanovllm/engine/model_runner.py does around the model on each
rank: runtime set-up between device selection and model construction (:26-31),
KV-cache allocation and binding (:103-121), batch -> tensors for prefill and
decode (:123-188), CUDA-graph capture and replay for decode (:195-212,
:222-257) and teardown order (:50-59).  The scheduler, block manager,
tokenizer and the shared-memory RPC between ranks stay outside: callers hand
in token lists and block tables (every rank must be given the same batch).
"""
from __future__ import annotations

from collections import Counter
from dataclasses import dataclass, field

import numpy as np
import torch
import torch.distributed as dist

from .. import ops
from ..layers.sampler import Sampler
from ..models.qwen3 import Qwen3ForCausalLM
from ..runtime import get_runtime, init_runtime, shutdown_runtime
from ..utils.context import reset_context, set_context

_TORCH_DTYPE = {np.dtype(np.int64): torch.int64, np.dtype(np.int32): torch.int32, np.dtype(np.float32): torch.float32}

FUSED_SAMPLER_MAX_ROWS = 256  # b2_lm_head_sample takes one token tile of the feature-lane layout


@dataclass
class ModelConfig:
    """The fields of a HF Qwen3 config the model reads (nanovllm/models/qwen3.py:127-143,167-171,199-203)."""
    hidden_size: int
    num_attention_heads: int
    num_key_value_heads: int
    head_dim: int
    intermediate_size: int
    num_hidden_layers: int
    vocab_size: int
    rms_norm_eps: float = 1e-6
    rope_theta: float = 1e6
    max_position_embeddings: int = 40960
    tie_word_embeddings: bool = False
    attention_bias: bool = False
    hidden_act: str = "silu"
    rope_scaling: dict | None = None


QWEN3_0_6B = dict(hidden_size=1024, num_attention_heads=16, num_key_value_heads=8, head_dim=128, intermediate_size=3072,
                  num_hidden_layers=28, vocab_size=151936, tie_word_embeddings=True)
QWEN3_8B = dict(hidden_size=4096, num_attention_heads=32, num_key_value_heads=8, head_dim=128, intermediate_size=12288,
                num_hidden_layers=36, vocab_size=151936, tie_word_embeddings=False)
QWEN3_32B = dict(hidden_size=5120, num_attention_heads=64, num_key_value_heads=8, head_dim=128, intermediate_size=25600,
                 num_hidden_layers=64, vocab_size=151936, tie_word_embeddings=False)


@dataclass
class Seq:
    """Minimal per-request state: the token ids so far, the KV blocks they
    occupy and how many leading tokens are already in the cache."""
    token_ids: list[int]
    block_table: list[int] = field(default_factory=list)
    num_cached_tokens: int = 0

    def __len__(self):
        return len(self.token_ids)


def random_init_(model: torch.nn.Module, seed: int, tp_rank: int) -> None:
    """Seeded N(0, 0.02) weights generated on the device (norm weights stay 1).
    Each rank draws its own shard: enough for throughput runs, where only the
    shapes matter; parity tests load shards of one full model instead."""
    g = torch.Generator(device="cuda").manual_seed(seed * 1000 + tp_rank)
    for name, p in model.named_parameters():
        if "norm" in name:
            p.data.fill_(1.0)
        else:
            p.data.copy_(torch.empty(p.shape, dtype=torch.float32, device=p.device).normal_(0, 0.02, generator=g))


_ROW_INPUT_BYTES = 28


def _row_inputs(buf: torch.Tensor) -> dict[str, torch.Tensor]:
    """The per-row inputs of a decode step as views of one byte buffer of _ROW_INPUT_BYTES per row."""
    n, out, at = buf.numel() // _ROW_INPUT_BYTES, {}, 0
    for name, dtype in (("input_ids", torch.int64), ("positions", torch.int64), ("slot_mapping", torch.int32),
                        ("context_lens", torch.int32), ("temperatures", torch.float32)):
        size = n * dtype.itemsize
        out[name] = buf[at:at + size].view(dtype)
        at += size
    return out


class ModelRunner:

    def __init__(self, config: ModelConfig, *, max_num_seqs: int = 512, max_model_len: int = 4096, max_num_batched_tokens: int = 16384,
                 kvcache_block_size: int = 256, num_kvcache_blocks: int | None = None, gpu_memory_utilization: float = 0.9,
                 enforce_eager: bool = False, oneshot_tokens: int = 1024, timeout_ms: int = 5000, seed: int = 0,
                 full_weights: dict | None = None, fused_sampler: bool | None = None, sample_seed: int = 0):
        assert dist.is_initialized(), "create the process group first (world size 1 included), as the reference does"
        self.config = config
        self.rank, self.world = dist.get_rank(), dist.get_world_size()
        self.block_size = kvcache_block_size
        self.max_num_seqs, self.max_model_len, self.max_num_batched_tokens = max_num_seqs, max_model_len, max_num_batched_tokens
        self.enforce_eager = enforce_eager
        # LM head and sampler in one pass (no [B, vocab] logits, no gather): the default at every world size
        if fused_sampler is None:
            fused_sampler = True
        self.fused_sampler = fused_sampler
        self.sample_seed = sample_seed
        self.device = torch.device("cuda", torch.cuda.current_device())
        # symmetric buffers exist before the layers are built, so graph capture sees fixed addresses
        self.runtime = init_runtime(max_tokens=max_num_batched_tokens, hidden=config.hidden_size, oneshot_tokens=oneshot_tokens,
                                    vocab=config.vocab_size, max_seqs=max_num_seqs, timeout_ms=timeout_ms)
        prev_dtype = torch.get_default_dtype()
        torch.set_default_dtype(torch.bfloat16)
        try:
            with self.device:  # (torch.set_default_device would leave a Python hook on every later torch call of the process)
                self.model = Qwen3ForCausalLM(config)
                if full_weights is not None:
                    self.model.load_full_weights(full_weights)
                else:
                    random_init_(self.model, seed, self.rank)
                self.sampler = Sampler()
                self._allocate_kv_cache(num_kvcache_blocks, gpu_memory_utilization)
                self.graphs: dict[int, torch.cuda.CUDAGraph] = {}
                if not enforce_eager:
                    self._capture_graphs()
        finally:
            torch.set_default_dtype(prev_dtype)

    # ---- teardown (reference :50-59) --------------------------------------
    def exit(self):
        self.graphs = {}
        self.graph_pool = None
        torch.cuda.synchronize()
        shutdown_runtime()

    # ---- KV cache (reference :103-121) -------------------------------------
    def _allocate_kv_cache(self, num_blocks: int | None, utilization: float):
        c = self.config
        self.num_kv_heads = c.num_key_value_heads // self.world
        block_bytes = 2 * c.num_hidden_layers * self.block_size * self.num_kv_heads * c.head_dim * 2
        if num_blocks is None:
            free, total = torch.cuda.mem_get_info()
            budget = int(total * utilization) - (total - free)
            # activations of the largest prefill step: a few [tokens, widest layer output] bf16 tensors
            widest = max(2 * c.intermediate_size // self.world, c.hidden_size, (c.num_attention_heads + 2 * c.num_key_value_heads) * c.head_dim // self.world)
            budget -= 6 * self.max_num_batched_tokens * widest * 2
            num_blocks = budget // block_bytes
        assert num_blocks > 0, "no memory left for the KV cache"
        self.num_kvcache_blocks = int(num_blocks)
        self.kv_cache = torch.zeros(2, c.num_hidden_layers, self.num_kvcache_blocks, self.block_size, self.num_kv_heads, c.head_dim,
                                    dtype=torch.bfloat16, device=self.device)
        for i, layer in enumerate(self.model.model.layers):
            layer.self_attn.attn.k_cache = self.kv_cache[0, i]
            layer.self_attn.attn.v_cache = self.kv_cache[1, i]

    # ---- batch -> tensors -----------------------------------------------------
    def _h2d(self, values, dtype):
        return torch.tensor(values, dtype=dtype, pin_memory=True).to(self.device, non_blocking=True)

    def _to_device(self, *arrays: np.ndarray) -> list[torch.Tensor]:
        """The arrays on the device, sent as one pinned buffer in one copy (a copy costs the host and the stream a few
        microseconds however small it is).  torch's pinned pool keeps the buffer until the copy has run."""
        offsets, size = [], 0
        for a in arrays:
            offsets.append(size)
            size += (a.nbytes + 15) & ~15
        host = torch.empty(max(size, 16), dtype=torch.uint8, pin_memory=True)
        raw = host.numpy()
        for a, off in zip(arrays, offsets):
            raw[off:off + a.nbytes] = a.reshape(-1).view(np.uint8)
        dev = host.to(self.device, non_blocking=True)
        return [dev[off:off + a.nbytes].view(_TORCH_DTYPE[a.dtype]).view(a.shape) for a, off in zip(arrays, offsets)]

    def _block_tables(self, seqs: list[Seq]) -> np.ndarray:
        width = max(len(s.block_table) for s in seqs)
        tables = np.full((len(seqs), width), -1, dtype=np.int32)
        for row, s in zip(tables, seqs):
            row[:len(s.block_table)] = s.block_table
        return tables

    def prepare_prefill(self, seqs: list[Seq], num_new: list[int] | None = None):
        """Tokens [num_cached, num_cached + new) of each sequence are computed;
        their K/V go to the slots their block table assigns (reference :129-170)."""
        bs = self.block_size
        starts = [s.num_cached_tokens for s in seqs]
        ends = [len(s) if num_new is None else a + num_new[i] for i, (s, a) in enumerate(zip(seqs, starts))]
        news = [b - a for a, b in zip(starts, ends)]
        total = sum(news)
        ids, pos = np.empty(total, dtype=np.int64), np.empty(total, dtype=np.int64)
        slots = np.empty(total, dtype=np.int32)
        used, at = 0, 0  # tokens with a slot, tokens so far
        for s, a, b, n in zip(seqs, starts, ends, news):
            ids[at:at + n] = s.token_ids[a:b]
            pos[at:at + n] = p = np.arange(a, b)
            if s.block_table:
                slots[used:used + n] = np.asarray(s.block_table, dtype=np.int32)[p // bs] * bs + p % bs
                used += n
            at += n
        cu_q, cu_k = np.zeros(len(seqs) + 1, dtype=np.int32), np.zeros(len(seqs) + 1, dtype=np.int32)
        np.cumsum(news, out=cu_q[1:])
        np.cumsum(ends, out=cu_k[1:])
        arrays = [ids, pos, cu_q, cu_k, cu_q[1:] - 1, slots[:used]]
        if cu_k[-1] > cu_q[-1]:
            arrays.append(self._block_tables(seqs))
        ids_t, pos_t, cu_q_t, cu_k_t, last_t, slots_t, *tables_t = self._to_device(*arrays)
        set_context(True, cu_q_t, cu_k_t, max(news), max(ends), slots_t if used else None, None, tables_t[0] if tables_t else None,
                    last_token_index=last_t)
        return ids_t, pos_t

    def prepare_decode(self, seqs: list[Seq]):
        """One new token per sequence: the last one of its list (reference :172-188)."""
        bs = self.block_size
        lens = [len(s) for s in seqs]
        ids_t, pos_t, slots_t, lens_t, tables_t = self._to_device(
            np.array([s.token_ids[-1] for s in seqs], dtype=np.int64), np.array([n - 1 for n in lens], dtype=np.int64),
            np.array([s.block_table[(n - 1) // bs] * bs + (n - 1) % bs for s, n in zip(seqs, lens)], dtype=np.int32),
            np.array(lens, dtype=np.int32), self._block_tables(seqs))
        set_context(False, slot_mapping=slots_t, context_lens=lens_t, block_tables=tables_t)
        return ids_t, pos_t

    # ---- forward ---------------------------------------------------------------
    @torch.inference_mode()
    def run_model(self, input_ids: torch.Tensor, positions: torch.Tensor, is_prefill: bool):
        return self.model.compute_logits(self.run_hidden(input_ids, positions, is_prefill))

    def run_hidden(self, input_ids: torch.Tensor, positions: torch.Tensor, is_prefill: bool):
        """The model forward up to the final norm (eager for prefill, a graph replay for decode)."""
        from ..utils.context import get_context
        n = input_ids.size(0)
        if is_prefill or self.enforce_eager or n > self.graph_bs[-1]:
            return self.model(input_ids, positions)
        ctx = get_context()
        bs = next(b for b in self.graph_bs if b >= n)
        gv = self.graph_vars
        gv["input_ids"][:n] = input_ids
        gv["positions"][:n] = positions
        gv["slot_mapping"].fill_(-1)  # padded rows store nothing
        gv["slot_mapping"][:n] = ctx.slot_mapping
        gv["context_lens"].zero_()
        gv["context_lens"][:n] = ctx.context_lens
        gv["block_tables"][:n, :ctx.block_tables.size(1)] = ctx.block_tables
        self._bt_rows = {}  # the graph's table no longer matches what _decode_graph_step last staged
        self.graphs[bs].replay()
        return gv["outputs"][:n]

    def _decode_staging(self):
        """Pinned host mirrors of the graphs' input buffers, allocated once: a decode step fills them with
        numpy and issues one asynchronous copy for all the per-row inputs straight into the graph's inputs (no per-step
        pinned allocations, no device-to-device staging copies)."""
        if getattr(self, "_stage", None) is None:
            gv = self.graph_vars
            self._stage = torch.zeros(gv["rows"].shape, dtype=torch.uint8, pin_memory=True)
            self._stage_tables = torch.zeros(gv["block_tables"].shape, dtype=torch.int32, pin_memory=True)
            self._stage_np = {k: v.numpy() for k, v in _row_inputs(self._stage).items()}
            self._stage_np["block_tables"] = self._stage_tables.numpy()
            self._bt_rows = {}  # row of the staged block table -> the blocks last copied into the graph's table for it
        return self._stage_np

    @torch.inference_mode()
    def _decode_graph_step(self, seqs: list[Seq], temperatures: list[float] | None):
        """prepare_decode + the graph replay of run_model in one go, for batches a captured graph covers.  Returns the
        hidden rows and the temperatures on the device (None for greedy decoding)."""
        n = len(seqs)
        bs = next(b for b in self.graph_bs if b >= n)
        np_ = self._decode_staging()
        blk = self.block_size
        lens = [len(s) for s in seqs]
        np_["input_ids"][:n] = [s.token_ids[-1] for s in seqs]
        np_["positions"][:n] = [l - 1 for l in lens]
        np_["context_lens"][:n] = lens
        np_["context_lens"][n:bs] = 0          # padded rows attend to nothing ...
        np_["slot_mapping"][:n] = [s.block_table[(l - 1) // blk] * blk + (l - 1) % blk for s, l in zip(seqs, lens)]
        np_["slot_mapping"][n:bs] = -1         # ... and store nothing
        if temperatures is not None:
            np_["temperatures"][:n] = temperatures
        # block tables change only when a sequence takes a new block (every 256 tokens) or the batch changes: rows are
        # rewritten, and the table copied, only then
        bt = np_["block_tables"]
        rows = self._bt_rows
        width, dirty = 0, False
        for i, s in enumerate(seqs):
            t = s.block_table
            width = max(width, len(t))
            if rows.get(i) != t:
                bt[i, :len(t)] = t
                rows[i] = list(t)
                dirty = True
        gv = self.graph_vars
        gv["rows"].copy_(self._stage, non_blocking=True)
        if dirty:
            gv["block_tables"][:n, :width].copy_(self._stage_tables[:n, :width], non_blocking=True)
        self.graphs[bs].replay()
        set_context(False)  # the LM head only needs to know this is not a prefill step
        return gv["outputs"][:n], gv["temperatures"][:n] if temperatures is not None else None

    @torch.inference_mode()
    def step(self, seqs: list[Seq], is_prefill: bool, temperatures: list[float] | None = None, num_new: list[int] | None = None):
        """One forward pass + sampling on rank 0; the chosen token ids are
        returned on every rank.  temperatures=None means greedy (argmax)."""
        if not is_prefill and not self.enforce_eager and len(seqs) <= self.graph_bs[-1]:
            hidden, temps = self._decode_graph_step(seqs, temperatures)
        else:
            ids, pos = self.prepare_prefill(seqs, num_new) if is_prefill else self.prepare_decode(seqs)
            hidden = self.run_hidden(ids, pos, is_prefill)
            temps = None if temperatures is None else self._h2d(temperatures, torch.float32)
        if getattr(self, "_picked", None) is None or self._picked.numel() < len(seqs):
            self._picked = torch.zeros(max(len(seqs), self.max_num_seqs), dtype=torch.int64, device=self.device)
        picked = self._picked[:len(seqs)]  # one buffer for every step: rank 0's sampler fills it, the broadcast hands it to the others
        if self.fused_sampler and (len(seqs) <= FUSED_SAMPLER_MAX_ROWS or self.world == 1):
            # (several ranks exchange once per call, so they take one call or the unfused path)
            for i in range(0, len(seqs), FUSED_SAMPLER_MAX_ROWS):
                rows = slice(i, i + FUSED_SAMPLER_MAX_ROWS)
                self.model.sample_tokens(hidden, None if temps is None else temps[rows], self.sample_seed, out=picked[rows], rows=rows)
        else:
            logits = self.model.compute_logits(hidden)
            if self.rank == 0:
                picked = Sampler.greedy(logits) if temps is None else self.sampler(logits, temps)
        if self.world > 1:
            ops.broadcast_tokens(picked)  # rank 0's choice reaches every rank on the device
        tokens = picked.tolist()  # the step's synchronisation point
        reset_context()
        self.runtime.check_status()
        return tokens

    @torch.inference_mode()
    def verify(self, seqs: list[Seq], drafts: list[list[int]], parents: list[list[int]], rules: dict[str, torch.Tensor] | None = None) -> list[list[int]]:
        """One forward pass over a tree of drafted tokens per sequence (speculative decoding): node 0 is the sequence's last token, as in a
        decode step, and drafts[i][j] is node j + 1, whose parent is node parents[i][j] <= j.  Returns the greedy pick after every node, on every rank.  The
        block tables must have room for all nodes, of which there are at most max_num_seqs in all; keys and values of node j are left at place
        len(seq) - 1 + j.  Whoever keeps a path other than nodes 0, 1, 2, ... moves its nodes together in kv_cache first: node j of the path to place len(seq) - 1 + j.  rules: arguments of
        ops.adjust_logits that belong to the sequences (histories end before the last token: node 0 counts as part of every path) or,
        allowed_mask, to the nodes in their order; they are looked at on rank 0 only, whose error makes every rank raise."""
        if not (len(seqs) == len(drafts) == len(parents)) or any(len(d) != len(p) for d, p in zip(drafts, parents)):
            raise ValueError("a list of drafted tokens and of their parents for each sequence")
        if not seqs:
            return []
        counts = [len(d) + 1 for d in drafts]
        total, words = sum(counts), -(-max(counts, default=1) // 64)
        if total > self.max_num_seqs:
            raise ValueError(f"{total} nodes: at most max_num_seqs ({self.max_num_seqs}), the rows of the logits")
        ids, mask, at = np.empty(total, dtype=np.int64), np.zeros((total, words), dtype=np.uint64), 0
        for s, d, p in zip(seqs, drafts, parents):
            ids[at:at + len(d) + 1] = [s.token_ids[-1], *d]
            for j in range(len(d) + 1):
                if j > 0:
                    if not 0 <= p[j - 1] < j:
                        raise ValueError(f"node {j}: parent {p[j - 1]}")
                    mask[at + j] = mask[at + p[j - 1]]
                mask[at + j, j // 64] |= np.uint64(1 << (j % 64))
            at += len(d) + 1
        cached = np.array([len(s) - 1 for s in seqs], dtype=np.int32)
        wanted = cached + np.array(counts, dtype=np.int32)
        if any(n > len(s.block_table) * self.block_size for s, n in zip(seqs, wanted)):
            raise ValueError("the block tables have no room for the drafted tokens")
        if max(wanted) > self.max_model_len:
            raise ValueError(f"{max(wanted)} tokens: at most max_model_len ({self.max_model_len})")
        # the caller has dealt the blocks: the stack holds the ones that the nodes open, the first of them on top
        opened = [b for s, c, n in zip(seqs, cached, wanted) for b in s.block_table[-(-c // self.block_size):-(-n // self.block_size)]]
        ids_t, cached_t, wanted_t, tables_t, mask_t, stack_t, height_t = self._to_device(
            ids, cached, wanted, self._block_tables(seqs), mask.view(np.int64), np.array(opened[::-1], dtype=np.int32), np.array([len(opened)], dtype=np.int32))
        inputs = ops.batch_inputs(tables_t, cached_t, wanted_t, stack_t, height_t, self.block_size, self.num_kvcache_blocks * self.block_size, total, tree_mask=mask_t)
        set_context(False, inputs.cu_seqlens_q, inputs.cu_seqlens_k, max(counts), int(wanted.max()), inputs.slot_mapping, inputs.context_lens, tables_t, tree_mask=mask_t)
        try:
            logits = self.model.compute_logits(self.model(ids_t, inputs.positions))
            picked, failed = torch.zeros(total, dtype=torch.int64, device=self.device), None
            if self.rank == 0:
                try:
                    if rules:
                        logits = ops.adjust_logits(logits, **rules, cu_seqlens=inputs.cu_seqlens_q, draft_tokens=ids_t, tree_mask=mask_t, out=logits)
                    ops.argmax(logits, out=picked)
                except Exception as error:  # (the other ranks are on their way to the broadcast: they get a token that there is not)
                    failed = error
                    picked.fill_(self.config.vocab_size)
            if self.world > 1:
                ops.broadcast_tokens(picked)
            flat = picked.tolist()  # the step's synchronisation point
        finally:
            reset_context()
        self.runtime.check_status()
        if failed is not None:
            raise failed
        if flat[0] >= self.config.vocab_size:
            raise RuntimeError("rank 0 could not apply the step's rules or pick its tokens; its own error says why")
        ends = np.cumsum(counts)
        return [flat[e - c:e] for e, c in zip(ends, counts)]

    @torch.inference_mode()
    def beam_search(self, seqs: list[Seq], beams: int, max_new_tokens: int, free_blocks: list[int], *, eos_token: int | None = None,
                    rules: dict[str, torch.Tensor] | None = None) -> list[list[tuple[list[int], float]]]:
        """The `beams` continuations of each sequence with the largest sums of log-probabilities that a beam search finds, best first, as (tokens, sum), on every rank; fewer
        where there are no more.  A continuation has max_new_tokens, or fewer and ends in eos_token.  The prompts' block tables have room for their tokens, of which
        num_cached_tokens are in the cache and the others are computed first, in one pass; they may share full blocks, and no others.  free_blocks: what the search may use; for each sequence `beams` times the blocks that
        max_new_tokens fill behind the prompt's full blocks.  Afterwards these blocks, and those of the prompts that are not full, hold nothing of use.  rules: arguments of ops.adjust_logits
        other than the histories (which are the prompts and the beams' tokens), a row for each sequence; looked at on rank 0 only, whose error makes every rank raise."""
        bs, n, rows = self.block_size, len(seqs), len(seqs) * beams
        if not 1 <= beams <= 32 or max_new_tokens < 1:
            raise ValueError(f"{beams} beams, {max_new_tokens} new tokens: 1 to 32 beams, at least one token")
        if not seqs:
            return []
        if rows > min(self.max_num_seqs, 1024) or n > 512:
            raise ValueError(f"{n} sequences of {beams} beams: at most max_num_seqs ({self.max_num_seqs}) rows, 1024, of 512 sequences")
        lens, news = [len(s) for s in seqs], [len(s) - s.num_cached_tokens for s in seqs]
        if min(news) < 1 or sum(news) > self.max_num_batched_tokens:
            raise ValueError(f"{sum(news)} prompt tokens to compute: at least one of each sequence, at most max_num_batched_tokens ({self.max_num_batched_tokens})")
        if max(lens) + max_new_tokens > self.max_model_len:
            raise ValueError(f"{max(lens)} + {max_new_tokens} tokens: at most max_model_len ({self.max_model_len})")
        if any(l > len(s.block_table) * bs for l, s in zip(lens, seqs)):
            raise ValueError("the block tables have no room for the prompts")
        full = [l // bs for l in lens]  # blocks of the prompts that stay as they are: all beams share them
        needed = sum(beams * (-(-(l + max_new_tokens) // bs) - f) for l, f in zip(lens, full))
        if len(free_blocks) < needed:
            raise ValueError(f"{len(free_blocks)} free blocks: the search may need {needed}")
        used = Counter(b for s, l in zip(seqs, lens) for b in s.block_table[:-(-l // bs)])
        if len(set(free_blocks)) < len(free_blocks) or any(b in used for b in free_blocks) or not all(0 <= b < self.num_kvcache_blocks for b in (*free_blocks, *used)):
            raise ValueError("the free blocks must be blocks of the cache, each once, and none of the prompts'")
        if any(l % bs and used[s.block_table[f]] > 1 for s, l, f in zip(seqs, lens, full)):  # (the first beams write to it, and give it back)
            raise ValueError("prompts may share full blocks only")
        # The rows before the first selection: the prompt in the first of each sequence, the others empty.
        width, most = -(-(max(lens) + max_new_tokens) // bs), max(lens)
        tables, row_lens = np.full((n, beams, width), -1, dtype=np.int32), np.zeros((n, beams), dtype=np.int32)
        past, said = np.zeros((n, beams, most + max_new_tokens), dtype=np.int64), np.zeros((n, beams), dtype=np.int32)
        for i, (s, l) in enumerate(zip(seqs, lens)):
            tables[i, 0, :-(-l // bs)] = s.block_table[:-(-l // bs)]
            row_lens[i, 0] = said[i] = l
            past[i, :, :l] = s.token_ids
        stack = np.zeros(len(free_blocks) + n, dtype=np.int32)  # (the prompts' open blocks may come to it)
        stack[:len(free_blocks)] = free_blocks
        tables_t, lens_t, past_t, said_t, prompt_t, stack_t, height_t, first_t, prefix_t, cu_t = self._to_device(
            tables.reshape(rows, width), row_lens.reshape(rows), past.reshape(rows, -1), said.reshape(rows), np.repeat(np.array(lens, dtype=np.int32), beams), stack,
            np.array([len(free_blocks)], dtype=np.int32), np.array(full, dtype=np.int32), np.array(full, dtype=np.int32) * bs, np.arange(0, rows + 1, beams, dtype=np.int32))
        live, ended = torch.zeros(n, 1, device=self.device), None
        try:
            ids, pos = self.prepare_prefill(seqs)
            logits = self.model.compute_logits(self.model(ids, pos))
            for step in range(max_new_tokens):
                picks = self._select_beams(logits, live, beams, ended, eos_token, rules, past_t, said_t, prompt_t)
                live, ended = picks.scores, picks.finished
                state = ops.reorder_beams(picks.parents, tables_t, lens_t, stack_t, height_t, self.kv_cache, first_blocks=first_t, history=past_t, history_lens=said_t, tokens=picks.tokens)
                tables_t, past_t, said_t = state.block_tables, state.history, state.history_lens
                if step + 1 == max_new_tokens or bool((ended | (picks.parents < 0)).all()):
                    break
                # Every row takes a token, so that the rows stay where they are; those that have ended, or are empty, see nothing.
                inputs = ops.batch_inputs(tables_t, state.context_lens, state.context_lens + 1, stack_t, state.num_free, bs, self.num_kvcache_blocks * bs, rows)
                lens_t, height_t = inputs.context_lens, inputs.num_free
                seen = torch.where(ended.view(rows) | (state.context_lens == 0), 0, lens_t)
                set_context(False, slot_mapping=inputs.slot_mapping, context_lens=seen, block_tables=tables_t, cu_groups=cu_t, prefix_lens=prefix_t, max_group=beams)
                logits = self.model.compute_logits(self.model(picks.tokens.view(rows).clamp(min=0), inputs.positions))
            if self.world > 1:  # (rank 0's, as bits; the broadcast takes no negative values)
                bits = live.reshape(rows).view(torch.int32).to(torch.int64) + (1 << 31)
                ops.broadcast_tokens(bits)
                live = (bits - (1 << 31)).to(torch.int32).view(torch.float32).view(n, beams)
            scores, said_h, past_h = live.tolist(), said_t.view(n, beams).tolist(), past_t.view(n, beams, -1).tolist()
        finally:
            reset_context()
        self.runtime.check_status()
        return [[(past_h[i][b][l:said_h[i][b]], scores[i][b]) for b in range(beams) if scores[i][b] > float("-inf")] for i, l in enumerate(lens)]

    def _select_beams(self, logits, scores, picks, ended, eos_token, rules, past, said, prompt_lens) -> ops.BeamPicks:
        """ops.beam_select on rank 0, and its picks on every rank (the scores on rank 0 only).  The logits are of as many rows a sequence as there are scores."""
        n = scores.shape[0]
        failed, out = None, None
        if self.rank == 0:
            try:
                if rules:
                    each, rows = scores.shape[1], slice(None, None, picks // scores.shape[1])  # (before the first selection all rows of a sequence have the prompt)
                    logits = ops.adjust_logits(logits, **{name: x.repeat_interleave(each, 0) for name, x in rules.items()}, history=past[rows], history_lens=said[rows].contiguous(),
                                               prompt_lens=prompt_lens[rows].contiguous(), out=logits)
                out = ops.beam_select(logits, scores, picks, finished=ended, eos_token=eos_token)
            except Exception as error:  # (the other ranks are on their way to the broadcast: they get a beam that there is not)
                failed = error
        if self.world > 1:
            # (not negative, which the broadcast does not take: token and parent from 0 on; a parent is one of 32, which leaves bit 7 to say that there are no picks)
            packed = torch.full((n * picks,), 1 << 7, dtype=torch.int64, device=self.device)
            if out is not None:
                packed = ((out.tokens + 1 << 8) | (out.parents + 1 << 1) | out.finished).view(-1)
            ops.broadcast_tokens(packed)
            if self.rank != 0:
                if int(packed[0]) == 1 << 7:
                    raise RuntimeError("rank 0 could not apply the step's rules or select its beams; its own error says why")
                packed = packed.view(n, picks)
                out = ops.BeamPicks(torch.zeros(n, picks, device=self.device), (packed >> 1 & 63).to(torch.int32) - 1, (packed >> 8) - 1, (packed & 1).bool())
        if failed is not None:
            raise failed
        return out

    # ---- CUDA graphs (reference :222-257) -----------------------------------------
    @torch.inference_mode()
    def _capture_graphs(self):
        c = self.config
        max_bs = min(self.max_num_seqs, 512)
        max_blocks = (self.max_model_len + self.block_size - 1) // self.block_size
        dev = self.device
        rows = torch.zeros(max_bs * _ROW_INPUT_BYTES, dtype=torch.uint8, device=dev)
        gv = dict(
            rows=rows,  # the per-row inputs below, side by side: one copy fills them all
            **_row_inputs(rows),
            block_tables=torch.zeros(max_bs, max_blocks, dtype=torch.int32, device=dev),
            outputs=torch.zeros(max_bs, c.hidden_size, dtype=torch.bfloat16, device=dev),
        )
        gv["slot_mapping"].fill_(-1)
        self.graph_bs = [b for b in (1, 2, 4, 8) if b <= max_bs] + list(range(16, max_bs + 1, 16))
        self.graph_pool = None
        for bs in reversed(self.graph_bs):
            graph = torch.cuda.CUDAGraph()
            set_context(False, slot_mapping=gv["slot_mapping"][:bs], context_lens=gv["context_lens"][:bs], block_tables=gv["block_tables"][:bs])
            gv["outputs"][:bs] = self.model(gv["input_ids"][:bs], gv["positions"][:bs])  # warm-up (also runs the collectives once)
            with torch.cuda.graph(graph, self.graph_pool):
                gv["outputs"][:bs] = self.model(gv["input_ids"][:bs], gv["positions"][:bs])
            if self.graph_pool is None:
                self.graph_pool = graph.pool()
            self.graphs[bs] = graph
            torch.cuda.synchronize()
            reset_context()
        self.graph_vars = gv


class ResidentDecoder:
    """Decode steps that never leave the device: one CUDA graph holds the model
    forward, the LM head with its gather, the greedy pick on rank 0, the token
    broadcast to the other ranks and the computation of the next step's inputs
    (what nanovllm/engine/model_runner.py:172-188 and :195-212 do with a host
    round trip every step).  `load(seqs)` puts a batch on the device;
    `replay()` advances every sequence by one token."""

    @torch.inference_mode()
    def __init__(self, runner: ModelRunner, batch: int):
        from .. import ops
        assert not runner.enforce_eager and batch in runner.graphs, "batch must be one of the captured decode batch sizes"
        self.r, self.bs, self.ops = runner, batch, ops
        self.tokens = torch.zeros(batch, dtype=torch.int64, device=runner.device)
        gv = runner.graph_vars
        gv["slot_mapping"].fill_(-1)
        gv["context_lens"].zero_()
        before = ops._abi.launch_count()
        self._body()  # warm-up: also creates the logits view outside the capture
        self.kernels_per_step = ops._abi.launch_count() - before
        gv["slot_mapping"].fill_(-1)
        gv["context_lens"].zero_()
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph, runner.graph_pool):
            self._body()
        torch.cuda.synchronize()
        self.replays_left = 0  # nothing loaded yet

    @torch.inference_mode()
    def _body(self):
        r, bs, gv = self.r, self.bs, self.r.graph_vars
        set_context(False, slot_mapping=gv["slot_mapping"][:bs], context_lens=gv["context_lens"][:bs], block_tables=gv["block_tables"][:bs])
        hidden = r.model(gv["input_ids"][:bs], gv["positions"][:bs])
        if r.fused_sampler and bs <= FUSED_SAMPLER_MAX_ROWS:
            r.model.sample_tokens(hidden, None, r.sample_seed, out=self.tokens)  # greedy: rank 0 gets the picks
        else:
            logits = r.model.compute_logits(hidden)
            if r.rank == 0:
                self.ops.argmax(logits, self.tokens)
        if r.world > 1:
            self.ops.broadcast_tokens(self.tokens)
        self.ops.advance_decode(self.tokens, gv["input_ids"], gv["positions"], gv["context_lens"], gv["slot_mapping"],
                                gv["block_tables"][:bs], r.block_size, r.num_kvcache_blocks * r.block_size)
        reset_context()

    @torch.inference_mode()
    def load(self, seqs: list[Seq]) -> None:
        """The batch's state as prepare_decode would build it for the next step."""
        r, gv, n = self.r, self.r.graph_vars, len(seqs)
        assert n == self.bs
        bs = r.block_size
        width = max(len(s.block_table) for s in seqs)
        assert width <= gv["block_tables"].shape[1], "a block table is longer than max_model_len allows"
        assert all(len(s) <= len(s.block_table) * bs for s in seqs), "a sequence is longer than its block table"
        gv["input_ids"][:n] = r._h2d([s.token_ids[-1] for s in seqs], torch.int64)
        gv["positions"][:n] = r._h2d([len(s) - 1 for s in seqs], torch.int64)
        gv["context_lens"][:n] = r._h2d([len(s) for s in seqs], torch.int32)
        gv["slot_mapping"][:n] = r._h2d([s.block_table[(len(s) - 1) // bs] * bs + (len(s) - 1) % bs for s in seqs], torch.int32)
        r._bt_rows = {}  # the graph's table is rewritten here: _decode_graph_step must stage its rows again
        gv["block_tables"][:n].fill_(-1)  # columns past a sequence's own blocks: no room (the advance kernel freezes such a row)
        gv["block_tables"][:n, :width] = r._h2d([s.block_table + [-1] * (width - len(s.block_table)) for s in seqs], torch.int32)
        # replays until the first sequence has filled its last block: each replay stores the K/V of one more position
        self.replays_left = min(len(s.block_table) * bs - len(s) for s in seqs) + 1

    def replay(self) -> None:
        if self.replays_left <= 0:
            raise RuntimeError("ResidentDecoder.replay: a sequence has filled the blocks it was loaded with; load() a batch with more blocks")
        self.replays_left -= 1
        self.graph.replay()


def sequential_block_tables(lengths: list[int], block_size: int, first_block: int = 0, permutation: list[int] | None = None) -> list[list[int]]:
    """Block tables for sequences of the given (maximum) lengths, taking blocks
    in order from `first_block`, or from `permutation` (a shuffled free list)."""
    tables, nxt = [], first_block
    for n in lengths:
        need = (n + block_size - 1) // block_size
        ids = list(range(nxt, nxt + need))
        if permutation is not None:
            ids = [permutation[i] for i in ids]
        tables.append(ids)
        nxt += need
    return tables
