"""``LLMEngine``: the Python entry point, with the surface of inference_engine/engine.py:35-244 --
``LLMEngine(model, engine_config, dtype, load_tokenizer, verbose)``, ``add_request``, ``step``,
``generate`` returning ``RequestOutput(seq_id, prompt_len, output_ids, text, ttft, latency)``.

One step: schedule -> pack the batch (one host->device transfer) -> the model's step function
(a captured CUDA graph for pure-decode steps, eager otherwise) -> sample on the device -> one small
device->host read of the new tokens -> bookkeeping.  Sampling is inside the captured graph, so a
decode step is one transfer in, one graph launch, one transfer out.
"""
from __future__ import annotations

import contextlib
import os
import time
import weakref
from collections import deque
from dataclasses import dataclass, replace

import numpy as np
import torch

from ..cache.manager import RequestCache
from ..config import EngineConfig, load_config
from ..kernels import gemm_tc, ops
from ..kernels.attention import captured_context_bounds, sharing_pays, sharing_weight
from ..models.decoder import DecoderModel
from ..parts.base import Runtime
from ..sampling.params import SamplingParams
from ..sampling.rules import RuleBook, mask_words
from ..sampling.sampler import Sampler
from ..weights import read_model_folder
from .prefix import Prefix, shared_groups
from .runner import ModelRunner
from .scheduler import Scheduler
from .sequence import Sequence

ACTIVATION_RESERVE = 768 * 2 ** 20      # kept free for activations when sizing the cache (inference_engine/engine.py:51)


@dataclass
class RequestOutput:
    seq_id: int
    prompt_len: int
    output_ids: list
    text: str | None
    ttft: float | None          # seconds from arrival to the first generated token
    latency: float | None       # seconds from arrival to the end
    logprobs: list | None = None        # of the output's tokens, where the request asked for them


PENDING = -1          # in token_ids: a token that the step in flight is sampling


class _InFlight:
    """A launched step whose sampled tokens the host has not read yet.  ``sources``: (pinned row, count)
    in the order of ``seqs`` -- one entry, or two when the step ran as two graphs."""

    def __init__(self, seqs, places, ending, sources, logprob_sources, event):
        self.seqs, self.places, self.ending, self.sources, self.event = seqs, places, ending, sources, event
        self.logprob_sources = logprob_sources        # (pinned row or None, count), as ``sources``

    def tokens(self) -> list:
        out = []
        for row, n in self.sources:
            out += row[:n].tolist()
        return out

    def logprobs(self) -> list:
        out = []
        for row, n in self.logprob_sources:
            out += [None] * n if row is None else row[:n].tolist()
        return out


class _DeviceMemory:
    """Memory that a captured graph writes, for ``torch.as_tensor``: a view that does not own it.  A tensor that did would keep the graphs captured
    after this one from using the memory again, as they may: what one replay leaves is read before the next."""

    def __init__(self, t):
        self.__cuda_array_interface__ = dict(shape=tuple(t.shape), typestr="<f4", data=(t.data_ptr(), False), version=2)


class _DecodeGraph:
    def __init__(self, graph, layout, buffer, tokens, kernels, ctx, logits):
        self.graph, self.layout, self.buffer, self.tokens = graph, layout, buffer, tokens
        self.kernels = kernels        # kernels of this package inside the captured step
        self.ctx = ctx
        self.logits = torch.as_tensor(_DeviceMemory(logits), device=logits.device) if logits.numel() else logits      # what a replay leaves


def _nvtx_range(name):
    return torch.cuda.nvtx.range(name)


class LLMEngine:
    def __init__(self, model: str, engine_config: EngineConfig | None = None, dtype=torch.bfloat16,
                 load_tokenizer: bool = True, verbose: bool = True, device: str = "cuda:0"):
        if not torch.cuda.is_available():
            raise RuntimeError("LLMEngine needs a CUDA device: every operator is a CUDA kernel of this package")
        self.cfg = engine_config or EngineConfig()
        self.verbose = verbose
        if not os.path.isdir(model):
            raise FileNotFoundError(f"{model!r} is not a model folder (config.json + *.safetensors); "
                                    "downloading by name is not supported")
        self.device = torch.device(device)
        torch.cuda.set_device(self.device)
        self.model_cfg = load_config(model)
        spec = self.model_cfg.model_spec()
        self.cfg.max_model_len = min(self.cfg.max_model_len, spec.max_position)      # inference_engine/engine.py:42
        self.eos_token_id = spec.eos_token_id
        self.vocab_size = spec.vocab_size
        self.dtype = dtype
        rt = Runtime(self.device, dtype)
        self.model = DecoderModel(spec, read_model_folder(model), rt, where=model)
        torch.cuda.empty_cache()

        layout = self.model.cache_layout
        per_page = sum(layout.bytes_per_page(g, self.cfg.block_size, dtype) for g in range(len(layout.groups)))
        if self.cfg.num_blocks is not None:
            num_blocks = int(self.cfg.num_blocks)
        else:                                      # size the pool from the memory left after the weights
            free, _ = torch.cuda.mem_get_info(self.device)
            state = layout.bytes_per_state_slot() * (self.cfg.max_num_seqs + 1)
            kv_bytes = int((free - ACTIVATION_RESERVE - state) * self.cfg.kv_cache_memory_fraction)
            num_blocks = kv_bytes // max(per_page, 1)
            # no request can use more than max_model_len positions: cap what max_num_seqs can ever hold
            ceiling = self.cfg.max_num_seqs * (-(-self.cfg.max_model_len // self.cfg.block_size)) + 1
            num_blocks = min(num_blocks, ceiling + max(1, ceiling // 100) + 1)
        if num_blocks < 2:
            raise RuntimeError(f"not enough memory for the cache: {num_blocks} pages of {per_page} bytes")
        self.runner = ModelRunner(self.model, num_blocks, self.cfg.block_size, self.cfg.max_num_seqs)
        self.cache = self.runner.cache
        self.scheduler = Scheduler(self.cfg, self.cache)
        self.max_blocks_per_seq = -(-self.cfg.max_model_len // self.cfg.block_size)
        self.sampler = Sampler(self.device, self.cfg.seed)
        if verbose:
            print(f"[mini_inference_engine_b200] cache: {num_blocks} pages x {self.cfg.block_size} tokens = "
                  f"{num_blocks * self.cfg.block_size} tokens ({num_blocks * per_page / 2 ** 30:.2f} GiB)")

        self.tokenizer = None
        if load_tokenizer and any(os.path.isfile(os.path.join(model, f))
                                  for f in ("tokenizer.json", "tokenizer.model", "tokenizer_config.json")):
            from transformers import AutoTokenizer          # text in/out only; never on the token path
            self.tokenizer = AutoTokenizer.from_pretrained(model)

        most = max(self.cfg.max_num_batched_tokens, self.cfg.max_num_seqs, 256, *self.cfg.cuda_graph_batch_sizes)
        # the sampled tokens as the host sees them: two rows, taken in turns (step N's are read while step
        # N+1 runs); the sampling kernel writes them itself (pinned memory is addressable from the device)
        self._pinned_tokens = torch.zeros(2, most, dtype=torch.int32, pin_memory=True)
        # a prompt portion that runs as a graph of its own beside the decode graph leaves its token apart
        self._pinned_portion = torch.zeros(2, 8, dtype=torch.int32, pin_memory=True)
        self._portion_slot = most
        self._sampled = torch.zeros(most + 8, dtype=torch.int32, device=self.device)   # the last step's tokens, on the device
        self._turn = 0
        self.rules = RuleBook(self.device, self.cfg.max_model_len, self.vocab_size)
        self._logprobs = self._pinned_logprobs = None        # made when a request first asks for them
        self.can_share = self.cache.can_share() and not layout.state         # whether requests can share pages
        self._host_state()
        self._shared_graphs: dict = {}           # (bucket, context bound) -> captured decode step over shared prefixes, or None: it has run once
        self._kv_shape = max(((n.num_kv_heads, n.head_dim) for _, n in layout.kv.values()), key=lambda s: s[0] * s[1], default=(0, 0))      # of the widest layer
        self.graphs: dict = {}                   # (bucket, context bound) -> captured decode step
        self.graph_sizes: list = []
        self.graph_bounds: list = []             # the context bounds the buckets were captured for, ascending
        self.num_steps = 0
        self.num_graph_steps = 0
        self.num_portion_graph_steps = 0
        self._portion_graphs: dict = {}          # (tokens, whether none of them pads, wanted logits, context bound) -> captured step of one prompt portion
        self._portion_seen: dict = {}
        self._graph_pool = None
        self._capture_stream = None
        self.h2d_bytes = 0
        self.d2h_bytes = 0
        if self.cfg.use_cuda_graphs:
            self._capture_cuda_graphs()
        if self.cfg.warm_up_prompt_step:
            self._warm_up_prompt_step()

    def _host_state(self) -> None:
        """What the host keeps between steps."""
        # (weakly: an engine that only the garbage collector could end might end, graphs and all, in the middle of another's capture)
        ended = weakref.WeakMethod(self._ended)

        def tell(seq):
            engine_hears = ended()
            if engine_hears is not None:
                engine_hears(seq)

        self.scheduler.ended = tell
        self._in_flight = None
        self._unreported: list = []              # requests that have ended and that no step has returned yet
        self._under_grammar: dict = {}           # live requests with a grammar, by id: a step without any looks at no request for it
        self.prefixes: list = []                 # the prefixes that requests may begin with (``add_prefix``)

    @torch.inference_mode()
    def _warm_up_prompt_step(self):
        """One prompt step of the whole token budget on scratch rows (tokens 0 at positions 0.. of page 0, as the
        padding of a portion graph; no logits wanted), and one that wants a token: what a first real step would
        otherwise pay for -- kernel modules loaded at first use, the library's choice of a product for that many rows,
        blocks of the allocator -- is paid here.  Nothing but the scratch page is written."""
        from .batch import BatchRow
        n = min(self.cfg.max_num_batched_tokens, self.cfg.max_model_len)
        if n < 2:
            return
        b = self.runner.builder
        pages = -(-n // self.cfg.block_size)
        zeros = [np.zeros(pages, dtype=np.int32) for _ in range(b.num_groups)]
        for want in ((), (n - 1,)):
            row = BatchRow(np.zeros(n, dtype=np.int32), 0, zeros, 0, want)
            buf, layout = b.pack([row], extras=self.sampler.inputs(len(want)))
            ctx = b.to_device(buf, layout)
            ctx.token_feedback = self._sampled
            self._forward_and_sample(ctx, self._sampled[self._portion_slot:self._portion_slot + len(want)],
                                     host_out=self._pinned_portion)
        torch.cuda.synchronize()

    # ------------------------------------------------------------------ CUDA graphs of decode steps
    def _forward_and_sample(self, ctx, tokens_out=None, host_out=None, seed=None):
        """Returns the step's logits; the tokens go to ``tokens_out``."""
        logits = self.model.step(ctx)
        if logits.shape[0]:
            self.sampler.sample(logits, ctx.extras["temperature"], ctx.extras["request"],
                                ctx.extras["out_position"], out=tokens_out, seed=seed,
                                host_out=self._pinned_tokens if host_out is None else host_out,
                                host_turn=ctx.extras["host_turn"])
        return logits

    def _choose_under_rules(self, seqs, logits, extras, at: int, turn: int, host_out):
        """The tokens of ``seqs`` once more where some have rules, chosen from a step's logits under them: over the tokens that the step itself chose.
        ``at``: the rows' first place among the sampled tokens.  Returns the pinned row that receives the log-probabilities, or None."""
        if not any(s.has_rules for s in seqs):
            return None
        k = len(seqs)
        lp = None
        if any(s.params.logprobs for s in seqs):
            if self._logprobs is None:
                self._logprobs = torch.zeros(self._sampled.numel(), dtype=torch.float32, device=self.device)
                self._pinned_logprobs = torch.zeros(2, self._sampled.numel(), dtype=torch.float32, pin_memory=True)
            lp = self._logprobs[at:at + k]
        tokens = self._sampled[at:at + k]
        if not self.sampler.sample_ruled(logits[:k], extras, tokens, seqs, self.rules, host_out=host_out, logprob=lp):
            host_out[turn, :k].copy_(tokens, non_blocking=True)
        if lp is None:
            return None
        row = self._pinned_logprobs[turn, at:at + k]
        row.copy_(lp, non_blocking=True)
        return row

    @torch.inference_mode()
    def _capture_cuda_graphs(self):
        """One graph per batch-size bucket, largest first so the smaller ones share its memory
        pool (inference_engine/engine.py:76-104), and per context bound (``graph_context_bounds``, those that the
        attention kernels of the compute type ask for, and ``max_model_len``): a step replays the graph of the smallest bound that covers its longest
        request.  A graph covers the whole step including the sampling kernel; its inputs live in one
        static device buffer that a step overwrites with one copy.  Rows that pad a batch up to its
        bucket are scratch rows: one token at position 0 of page 0, context length 1."""
        t0 = time.perf_counter()
        sizes = sorted(b for b in self.cfg.cuda_graph_batch_sizes if b <= self.cfg.max_num_seqs)
        if not sizes:
            return
        b = self.runner.builder
        pool = None
        asked = {*self.cfg.graph_context_bounds, *captured_context_bounds(self.dtype)}
        bounds = sorted({c for c in asked if c < self.cfg.max_model_len} | {self.cfg.max_model_len})
        for bs in reversed(sizes):
            static = None
            for bound in reversed(bounds):
                buf, layout = b.pack([], pad_rows=bs, table_width=self.max_blocks_per_seq,
                                     extras=self.sampler.inputs(bs))
                layout["max_ctx_len"] = bound                       # static bound for kernels that plan by it
                if static is None:                                  # the bounds of a bucket share its input buffer
                    static = torch.zeros(layout["size"], dtype=torch.int32, device=self.device)
                ctx = b.to_device(buf, layout, into=static)
                ctx.token_feedback = self._sampled
                tokens = self._sampled[:bs]
                self._forward_and_sample(ctx, tokens)               # warm-up: builds kernels, sizes buffers
                torch.cuda.synchronize()
                g = torch.cuda.CUDAGraph()
                before = ops.launches
                with torch.cuda.graph(g, pool=pool):
                    logits = self._forward_and_sample(ctx, tokens)
                pool = g.pool()
                self.graphs[bs, bound] = _DecodeGraph(g, layout, static, tokens, ops.launches - before, ctx, logits)
                del logits                                          # (its memory goes to the graphs behind)
        torch.cuda.synchronize()
        self._graph_pool = pool
        self.graph_sizes = sizes
        self.graph_bounds = bounds
        if self.verbose:
            print(f"[mini_inference_engine_b200] captured {len(self.graphs)} decode graphs (batch <= {sizes[-1]}, "
                  f"contexts <= {' / '.join(str(c) for c in bounds)}) in {time.perf_counter() - t0:.1f} s")

    def decode_graph(self, rows: int, context: int):
        """The captured step that serves ``rows`` decoding requests whose longest context (the new token
        included) is ``context``."""
        bs = next(s for s in self.graph_sizes if s >= rows)
        return self.graphs[bs, next(c for c in self.graph_bounds if c >= context)]

    # ------------------------------------------------------------------ CUDA graphs of decode steps over shared prefixes
    SHARED_GROUPS = 8        # prefixes that the rows of a step may share between them; with more, every row reads all of its pages itself

    def _shared_step(self, dseqs):
        """The groups of decoding rows that share a prefix, if the step is to read those once a group; else None."""
        if self.dtype != torch.bfloat16:
            return None
        groups = shared_groups(dseqs, self.cfg.block_size)
        if not groups or len(groups) > self.SHARED_GROUPS:
            return None
        heads, head_dim = self._kv_shape
        per_key = 2 * 2 * heads * head_dim
        own = sum(s.cache.num_computed + 1 for s in dseqs) - sum(n * positions for n, _, positions in groups)
        weight = sharing_weight(head_dim, heads, len(dseqs), own * per_key, sum(positions for _, _, positions in groups) * per_key)
        return groups if sharing_pays(groups, per_key, weight) else None

    def _decode_shared(self, drows, extras, groups, context: int):
        """Runs a decode step whose rows share prefixes: from its bucket's graph, which is captured the second time the bucket occurs (the first time
        builds kernels and sizes buffers).  Returns (extras on the device, logits)."""
        b = self.runner.builder
        bs = next(s for s in self.graph_sizes if s >= len(drows))
        bound = next(c for c in self.graph_bounds if c >= context)
        buf, layout = b.pack(drows, pad_rows=bs, table_width=self.max_blocks_per_seq, extras=extras, shared=groups, most_groups=self.SHARED_GROUPS)
        layout["max_ctx_len"] = bound
        self.h2d_bytes += buf.nbytes
        tokens = self._sampled[:bs]
        seen, g = (bs, bound) in self._shared_graphs, self._shared_graphs.get((bs, bound))
        if not seen:
            ctx = b.to_device(buf, layout)
            ctx.token_feedback = self._sampled
            logits = self._forward_and_sample(ctx, tokens)
            self._shared_graphs[bs, bound] = None
            return ctx.extras, logits
        if g is None:
            static = torch.zeros(layout["size"], dtype=torch.int32, device=self.device)
            ctx = b.to_device(buf, layout, into=static)
            ctx.token_feedback = self._sampled
            graph = torch.cuda.CUDAGraph()
            before = ops.launches
            with self._capturing(graph):
                logits = self._forward_and_sample(ctx, tokens)
            if self._graph_pool is None:
                self._graph_pool = graph.pool()
            g = self._shared_graphs[bs, bound] = _DecodeGraph(graph, layout, static, tokens, ops.launches - before, ctx, logits)
            del logits
        assert layout["size"] == g.layout["size"]
        b.to_device(buf, g.layout, into=g.buffer)
        g.graph.replay()
        self.num_graph_steps += 1
        return g.ctx.extras, g.logits

    # ------------------------------------------------------------------ CUDA graphs of prompt portions
    PORTION_GRAPH_MIN_TOKENS = 2

    @contextlib.contextmanager
    def _capturing(self, graph):
        """Captures what the body launches into ``graph`` (memory from the graphs' shared pool) in the middle of
        serving: on a side stream that waits for the serving stream, without the device-wide synchronisation and the
        emptying of the device and pinned-memory caches that ``torch.cuda.graph`` begins with -- those cost a capture
        10 to 60 ms, stall the step in flight, and leave the next eager steps to allocate their buffers anew."""
        if self._capture_stream is None:
            self._capture_stream = torch.cuda.Stream(device=self.device)
        side, main = self._capture_stream, torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            graph.capture_begin(self._graph_pool) if self._graph_pool is not None else graph.capture_begin()
            try:
                yield
            finally:
                graph.capture_end()
        main.wait_stream(side)

    @staticmethod
    def _padded_length(n: int) -> int:
        """The token count of the graph that serves a portion of ``n`` tokens: the next multiple of 32 up to
        256 tokens, of 64 up to 1,024, of 128 beyond (at most an eighth more tokens than the portion has)."""
        step = 32 if n <= 256 else (64 if n <= 1024 else 128)
        return -(-n // step) * step

    def _portion_rows(self, row, padded: int):
        """The portion's row and, behind it, a scratch row that brings the batch to ``padded`` tokens: its
        tokens sit at positions 0.. of page 0 (every block-table entry 0, state slot 0), nobody wants their
        logits, and what they write lands in the scratch page."""
        from .batch import BatchRow
        extra = padded - len(row.tokens)
        if extra == 0:
            return [row]
        pages = -(-extra // self.cfg.block_size)
        zeros = [np.zeros(pages, dtype=np.int32) for _ in row.tables]
        return [row, BatchRow(np.zeros(extra, dtype=np.int32), 0, zeros, 0, ())]

    @torch.inference_mode()
    def _portion_graph(self, row, extras, wanted: int):
        """The captured step for ONE prompt portion, if a step of the same padded shape (tokens, wanted
        logits) has run before; else None, and the shape is remembered.  Launching some 160 kernels one by
        one costs the host about 3 ms a step, more than a short portion takes on the device; portions are
        cut by what is left of the token budget, so their lengths are rounded up (``_padded_length``) for
        shapes to repeat.  What differs between replays -- tokens, positions, block table, the split between
        the portion and its padding, sampling inputs -- lives in the graph's static input buffer; the context
        bound that kernels plan by is the model's longest, or a shorter one that the attention kernels of the
        compute type ask for (a graph of its own).  At most ``graph_prompt_portions`` graphs are kept
        (the least recently used one goes).  The reference launches such steps eagerly."""
        n = len(row.tokens)
        padded = self._padded_length(n)
        longest = self.cfg.max_model_len
        bound = min((c for c in captured_context_bounds(self.dtype) if c >= row.pos0 + n), default=longest)
        key = (padded, padded == n, wanted, min(bound, longest))
        g = self._portion_graphs.get(key)
        if g is not None:
            self._portion_graphs[key] = self._portion_graphs.pop(key)        # most recently used last
            return g
        if not self._portion_seen.get(key):
            if len(self._portion_seen) > 256:
                self._portion_seen.clear()
            self._portion_seen[key] = 1
            return None
        b = self.runner.builder
        buf, layout = b.pack(self._portion_rows(row, padded), table_width=self.max_blocks_per_seq, extras=extras)
        layout["max_ctx_len"] = key[3]
        layout["q_len"] = None              # the split between portion and padding changes from replay to replay
        layout["few_single_rows"] = True    # (a padding of one token is a row like a decoding one: the kernel for portions serves it)
        static = torch.zeros(layout["size"], dtype=torch.int32, device=self.device)
        ctx = b.to_device(buf, layout, into=static)
        ctx.token_feedback = self._sampled
        tokens = self._sampled[self._portion_slot:self._portion_slot + wanted]
        # no warm-up run: a step of this padded length has run before, eagerly and unpadded, so nearly all kernels are built and loaded
        # (one that only the padded length takes sets itself up inside the capture, which the libraries allow for), and running
        # this one twice would write the request's cache twice -- harmless, but not free
        graph = torch.cuda.CUDAGraph()
        before = ops.launches
        with self._capturing(graph):
            logits = self._forward_and_sample(ctx, tokens, host_out=self._pinned_portion)
        if self._graph_pool is None:
            self._graph_pool = graph.pool()
        g = _DecodeGraph(graph, layout, static, tokens, ops.launches - before, ctx, logits)
        del logits
        while len(self._portion_graphs) >= max(1, self.cfg.graph_prompt_portions):
            self._portion_graphs.pop(next(iter(self._portion_graphs)))
        self._portion_graphs[key] = g
        return g

    # ------------------------------------------------------------------ requests
    def _prompt_ids(self, prompt) -> list:
        if isinstance(prompt, str):
            if self.tokenizer is None:
                raise ValueError("a text prompt needs a tokenizer in the model folder; pass token ids instead")
            ids = self.tokenizer.encode(prompt)
        else:
            ids = [int(t) for t in prompt]
        if not ids:
            raise ValueError("empty prompt")
        bad = [t for t in ids if not 0 <= t < self.vocab_size]
        if bad:
            raise ValueError(f"token id {bad[0]} is outside the vocabulary [0, {self.vocab_size})")
        return ids

    @torch.inference_mode()
    def add_prefix(self, prompt) -> Prefix:
        """Computes the keys and values of ``prompt`` (as many of its tokens as fill whole pages) once, for requests that begin with it
        (``add_request(..., prefix=)``): they share the pages, and steps in which many rows share them read them once (``generate``).  The pages are held until
        ``release_prefix``.  Refused with ValueError where a layer keeps a window, a block of positions or a state, and where the
        pages would leave a request that waits or runs too few ever to end."""
        ids = self._prompt_ids(prompt)
        pages = len(ids) // self.cfg.block_size
        if not self.can_share:
            raise ValueError("requests of this model cannot share pages: a layer keeps a window, a block of positions or a state per request")
        if not pages:
            raise ValueError(f"a prefix of {len(ids)} tokens fills no page of {self.cfg.block_size}")
        if len(ids) > self.cfg.max_model_len:
            raise ValueError(f"prefix of {len(ids)} tokens exceeds max_model_len {self.cfg.max_model_len}")
        refused = self._no_room_for_prefix(pages)
        if refused:
            raise ValueError(refused)
        p = Prefix(ids[:pages * self.cfg.block_size])
        try:
            self._compute_prefix(p)
        except BaseException:
            self.cache.free(p.cache)
            raise
        self.cache.pin(p.cache)
        self.prefixes.append(p)
        return p

    def _no_room_for_prefix(self, pages: int) -> str | None:
        """Why a prefix of so many pages cannot be held now; None where it can."""
        for s in (*self.scheduler.running, *self.scheduler.waiting):
            if not self.scheduler.can_ever_fit(self._most_positions(s.prompt_len, s.params), s.prefix_pages, pinned=pages):
                return f"a prefix of {pages} pages would leave request {s.seq_id} too few"
        if not self.cache.can_reserve(RequestCache(), pages * self.cfg.block_size, watermark=self.scheduler.watermark):
            return f"a prefix of {pages} pages, {min(q.num_free for q in self.cache.pools)} free"
        return None

    def _compute_prefix(self, p: Prefix) -> None:
        arr = np.asarray(p.token_ids, dtype=np.int32)
        for a in range(0, arr.size, self.cfg.max_num_batched_tokens):
            part = arr[a:a + self.cfg.max_num_batched_tokens]
            self.cache.reserve(p.cache, part.size)
            ctx = self.runner.builder.build([self.runner.make_row(p.cache, part, ())])
            ctx.token_feedback = self._sampled
            self.model.step(ctx)
            self.cache.advance(p.cache, part.size)

    def release_prefix(self, prefix: Prefix) -> None:
        """No further request begins with ``prefix``; its pages go back when the last that does has ended."""
        if prefix not in self.prefixes:
            raise ValueError("not a prefix of this engine, or released already")
        prefix.closed = True
        self.prefixes.remove(prefix)
        if not prefix.users:
            self._free_prefix(prefix)

    def _free_prefix(self, prefix: Prefix) -> None:
        self.cache.pin(prefix.cache, False)
        self.cache.free(prefix.cache)

    def _ended(self, seq) -> None:
        """What a request that has ended, whoever ended it, holds beside its pages goes back (the scheduler calls it)."""
        self.rules.release(seq)
        self._under_grammar.pop(seq.seq_id, None)
        if seq.prefix is not None:
            prefix, seq.prefix = seq.prefix, None
            prefix.users -= 1
            if prefix.closed and not prefix.users:
                self._free_prefix(prefix)

    def _checked(self, prompt, params: SamplingParams | None) -> tuple:
        """A request's prompt and options as they are run; ValueError for those that are not taken."""
        ids = self._prompt_ids(prompt)
        params = params or SamplingParams()
        if params.logit_bias:                    # (a copy of its own: the device takes the list at the request's first token, and its length at every one)
            params = replace(params, logit_bias=dict(params.logit_bias))
            if max(params.logit_bias) >= self.vocab_size:
                raise ValueError(f"logit_bias names token {max(params.logit_bias)}, outside the vocabulary [0, {self.vocab_size})")
        if len(ids) > self.cfg.max_model_len:
            raise ValueError(f"prompt of {len(ids)} tokens exceeds max_model_len {self.cfg.max_model_len}")
        if len(ids) + params.max_tokens > self.cfg.max_model_len:     # inference_engine/engine.py:126-127
            params = replace(params, max_tokens=max(1, self.cfg.max_model_len - len(ids)))
        return ids, params

    def _most_positions(self, prompt_len: int, params: SamplingParams) -> int:
        return min(prompt_len + params.max_tokens, self.cfg.max_model_len)

    def _refuse_what_never_fits(self, prompt_len: int, params: SamplingParams, shared: int = 0) -> None:
        most = self._most_positions(prompt_len, params)
        if not self.scheduler.can_ever_fit(most, shared):
            raise ValueError(f"a request of {most} positions can never fit the cache "
                             f"({self.cache.pools[0].num_usable} usable pages of {self.cfg.block_size}, {self.cache.pinned[0]} held by prefixes)")

    def add_request(self, prompt, params: SamplingParams | None = None, prefix: Prefix | None = None) -> Sequence:
        """``prefix``: what the prompt begins with, from ``add_prefix``; the request shares its pages (all of them that lie in front of the prompt's
        last token)."""
        ids, params = self._checked(prompt, params)
        shared = 0
        if prefix is not None:
            if prefix not in self.prefixes:
                raise ValueError("not a prefix of this engine, or released already")
            shared = min(len(prefix.token_ids), len(ids) - 1) // self.cfg.block_size
            if ids[:len(prefix.token_ids)] != prefix.token_ids[:len(ids)]:
                raise ValueError("the prompt does not begin with the prefix")
        self._refuse_what_never_fits(len(ids), params, shared)
        seq = Sequence(ids, params)
        if shared:
            seq.prefix, seq.prefix_pages = prefix, shared
            prefix.users += 1
        if params.grammar is not None:
            self._under_grammar[seq.seq_id] = seq
        self.scheduler.add(seq)
        return seq

    # ------------------------------------------------------------------ grammars
    def _ask_grammars(self) -> None:
        """Before a step: what every live request's grammar allows next.  A grammar reads the tokens so far, so the step in flight is read first.  The requests
        that end here (their grammar allows nothing) are reported beside those that ended with the step that was read: by this step, or, where a
        grammar fails, by the next."""
        if not self._under_grammar:
            return
        self._unreported += self.drain()
        for s in tuple(self._under_grammar.values()):
            if s.mask_at == len(s.token_ids):
                continue
            try:
                s.mask = mask_words(s.params.grammar.allowed(list(s.output_ids)), self.vocab_size, s.params.banned())
            except BaseException:            # the request goes (the exception is its report), the others and the engine stay as they are
                self._end_now(s)
                raise
            s.mask_at = len(s.token_ids)
            if s.mask is not None and not s.mask.any():
                self._end_now(s)
                self._unreported.append(s)

    def _end_now(self, seq) -> None:
        seq.finish_time = time.perf_counter()
        self.scheduler.finish(seq)

    # ------------------------------------------------------------------ one engine step
    def has_work(self) -> bool:
        return self.scheduler.has_work() or self._in_flight is not None or bool(self._unreported)

    @torch.inference_mode()
    def step(self) -> list:
        """One scheduling + model step; returns the requests whose end became known in it.

        With ``overlap_steps`` the host runs one step ahead of the device: step N+1 is scheduled,
        packed and launched while step N still runs, and only then are step N's tokens read.  The
        tokens a step samples stay on the device and are fed to the next step there (a token id
        -(k+1) in the batch means "entry k of the previous step's samples"), so nothing but the stop
        rules waits for the host: a request that ends by count is known beforehand, one that ends by
        EOS runs one step too many, whose token is dropped."""
        self._ask_grammars()
        launched = self._launch()
        if self._in_flight is not None:
            self._unreported += self._complete(self._in_flight)
        self._in_flight = launched
        # nothing to run ahead of: read the step's tokens now (also keeps the reference's loop
        # `while engine.scheduler.has_work(): engine.step()` complete)
        if launched is not None and (not self.cfg.overlap_steps or not self.scheduler.has_work()):
            self._unreported += self.drain()
        finished, self._unreported = self._unreported, []
        return finished

    def drain(self) -> list:
        """Reads the tokens of the step in flight, if any; returns the requests that ended with it."""
        fl, self._in_flight = self._in_flight, None
        return self._complete(fl) if fl is not None else []

    def _launch(self):
        with _nvtx_range("schedule"):
            batch = self.scheduler.schedule()
        if not batch:
            return None
        with _nvtx_range("prepare"):
            if any(s.prefix is not None for s, _ in batch):    # rows of one prefix side by side (a stable sort: the rest keep their order)
                batch.sort(key=lambda e: (0, e[0].prefix.serial, e[0].cache.shared) if e[0].prefix is not None else (1, 0, 0))
            rows, sample_seqs, decoding, others = [], [], [], []
            make_row = self.runner.make_row
            for i, (seq, n) in enumerate(batch):
                nc = seq.cache.num_computed
                last = nc + n == len(seq.token_ids)
                if nc + n <= seq.prompt_len:
                    tokens = seq.prompt_array[nc:nc + n]       # a view: a prompt portion
                else:
                    tokens = seq.token_ids[nc:nc + n]
                    if tokens[-1] == PENDING:              # sampled by the step in flight: read on the device
                        tokens[-1] = -(seq.pending_index + 1)
                rows.append(make_row(seq.cache, tokens, (n - 1,) if last else ()))
                if last:
                    sample_seqs.append(seq)
                (decoding if n == 1 and last else others).append(i)
            turn = self._turn ^ 1                              # the row of the pinned token buffers that this step fills
            row_seeds, seeds = self.sampler.seeds_of(sample_seqs)
            graphs_ok = bool(self.graph_sizes) and len(decoding) <= self.graph_sizes[-1] and seeds <= {self.cfg.seed}
            use_graph = graphs_ok and not others
            # One prompt portion, alone or beside requests that decode, runs as a graph of its padded length
            # -- beside the decode bucket's graph if there is one: two replays instead of some 200 launches
            # that cost the host more than the step costs the device.  The rows of the two replays do not
            # depend on one another, so the split changes nothing in what each computes.
            portion_graph = (graphs_ok and self.cfg.use_cuda_graphs and self.cfg.graph_prompt_portions > 0
                             and len(others) == 1 and len(rows[others[0]].tokens) >= self.PORTION_GRAPH_MIN_TOKENS
                             and (not decoding or len(rows[others[0]].tokens) <= self.cfg.split_step_max_tokens))

        def extras_for(seqs, pad_to):
            return self.sampler.inputs(pad_to or len(seqs), seqs, turn)

        with _nvtx_range("forward"):
            b = self.runner.builder
            sources, logprob_sources = [], []
            sampled_for = []                                   # the requests of ``sources``' tokens, in their order: not always the batch's
            if use_graph or (portion_graph and decoding):      # ---- the requests that decode, from their bucket's graph
                drows = [rows[i] for i in decoding]
                dseqs = [batch[i][0] for i in decoding]
                bs = next(s for s in self.graph_sizes if s >= len(drows))
                context = max(seq.cache.num_computed + 1 for seq in dseqs)
                groups = self._shared_step(dseqs)
                if groups:
                    extras, logits = self._decode_shared(drows, extras_for(dseqs, bs), groups, context)
                else:
                    g = self.decode_graph(bs, context)
                    buf, layout = b.pack(drows, pad_rows=bs, table_width=self.max_blocks_per_seq, extras=extras_for(dseqs, bs))
                    assert layout["size"] == g.layout["size"]
                    b.to_device(buf, g.layout, into=g.buffer)
                    g.graph.replay()
                    self.h2d_bytes += buf.nbytes
                    extras, logits = g.ctx.extras, g.logits
                    if use_graph:
                        self.num_graph_steps += 1
                lp = self._choose_under_rules(dseqs, logits, extras, 0, turn, self._pinned_tokens)
                sources.append((self._pinned_tokens[turn], len(dseqs)))
                logprob_sources.append((lp, len(dseqs)))
                sampled_for += dseqs
                for k, seq in enumerate(dseqs):
                    seq.pending_index = k
            if use_graph:
                pass
            elif portion_graph:                                # ---- the one prompt portion, from a graph of its padded length
                row = rows[others[0]]
                pseq = batch[others[0]][0]
                pseqs = [pseq] if row.want else []
                extras = extras_for(pseqs, 0)
                pg = self._portion_graph(row, extras, len(pseqs))
                tokens = self._sampled[self._portion_slot:self._portion_slot + len(pseqs)]
                if pg is not None:
                    buf, layout = b.pack(self._portion_rows(row, self._padded_length(len(row.tokens))),
                                         table_width=self.max_blocks_per_seq, extras=extras)
                    assert layout["size"] == pg.layout["size"]
                    b.to_device(buf, pg.layout, into=pg.buffer)
                    pg.graph.replay()
                    self.num_portion_graph_steps += 1
                    ctx, logits = pg.ctx, pg.logits
                else:                                          # the first time a shape occurs: launched kernel by kernel
                    buf, layout = b.pack([row], extras=extras)
                    ctx = b.to_device(buf, layout)
                    ctx.token_feedback = self._sampled
                    logits = self._forward_and_sample(ctx, tokens, host_out=self._pinned_portion)
                self.h2d_bytes += buf.nbytes
                if pseqs:
                    lp = self._choose_under_rules(pseqs, logits, ctx.extras, self._portion_slot, turn, self._pinned_portion)
                    sources.append((self._pinned_portion[turn], 1))
                    logprob_sources.append((lp, 1))
                    sampled_for += pseqs
                    pseq.pending_index = self._portion_slot
            else:                                              # ---- any other mix: one batch, launched kernel by kernel
                k = len(sample_seqs)
                extras = extras_for(sample_seqs, 0)
                groups = self._shared_step([seq for seq, _ in batch]) if not others else None
                buf, layout = b.pack(rows, extras=extras, shared=groups)
                ctx = b.to_device(buf, layout)
                ctx.token_feedback = self._sampled
                self.h2d_bytes += buf.nbytes
                logits = self.model.step(ctx)
                lp = None
                if any(s.has_rules for s in sample_seqs):
                    lp = self._choose_under_rules(sample_seqs, logits, ctx.extras, 0, turn, self._pinned_tokens)
                elif sample_seqs and not self.sampler.sample_step(logits, ctx.extras, self._sampled[:k], row_seeds, seeds,
                                                                  host_out=self._pinned_tokens):
                    self._pinned_tokens[turn, :k].copy_(self._sampled[:k], non_blocking=True)   # this rare way copies
                sources.append((self._pinned_tokens[turn], k))
                logprob_sources.append((lp, k))
                sampled_for += sample_seqs
                for k2, seq in enumerate(sample_seqs):
                    seq.pending_index = k2
            self._turn = turn
            self.d2h_bytes += 4 * len(sample_seqs)             # written by the sampling kernel into pinned host memory
            done_event = torch.cuda.Event()
            done_event.record()

        ending = self._advance(batch, sampled_for)
        return _InFlight(sampled_for, [s.num_tokens - 1 for s in sampled_for], ending, sources, logprob_sources, done_event)

    def _advance(self, batch, sample_seqs) -> list:
        """Bookkeeping that does not need a launched step's tokens: progress, the place each token will take, and the requests that end by count
        with this step, which are returned."""
        self.num_steps += 1
        for seq, n in batch:
            self.cache.advance(seq.cache, n)
        ending = []
        max_len = self.cfg.max_model_len
        for seq in sample_seqs:
            seq.token_ids.append(PENDING)
            total = len(seq.token_ids)
            if total - seq.prompt_len >= seq.params.max_tokens or total >= max_len:
                self.scheduler.finish(seq)                 # its pages may go to the next step: that one runs after this one
                ending.append(seq)
        return ending

    def _complete(self, fl) -> list:
        with _nvtx_range("sample"):
            fl.event.synchronize()
            new_tokens, new_logprobs = fl.tokens(), fl.logprobs()
        ops.check_range_errors()           # an integer out of range that a kernel refused to follow
        ops.check_tc_errors()
        gemm_tc.check_error()              # a bounded wait that ran out in a tensor-core product is an error, not a result
        now = time.perf_counter()
        finished = []
        for seq, place, tok, lp in zip(fl.seqs, fl.places, new_tokens, new_logprobs):
            if seq.ended_by_eos:
                del seq.token_ids[place:]                  # it ended by EOS a step ago: this token is one too many
                continue
            seq.token_ids[place] = tok
            if seq.params.logprobs:
                seq.logprobs.append(lp)
            if seq.first_token_time is None:
                seq.first_token_time = now
            if seq in fl.ending:
                seq.finish_time = now
                finished.append(seq)
            elif tok == self.eos_token_id and not seq.params.ignore_eos:      # inference_engine/engine.py:222-224
                del seq.token_ids[place + 1:]              # a token pending from the step already in flight
                seq.ended_by_eos = True
                seq.finish_time = now
                self.scheduler.finish(seq)
                finished.append(seq)
        return finished

    # ------------------------------------------------------------------ offline API
    def _add_answers(self, asked: deque, n: int, seqs: list, arrival: float) -> None:
        """Adds ``n`` answers to each of the next prompts (``asked``, from the front), behind its pages, for as long as there are places for them and
        room for the pages beside the requests that live.  With no request alive there is: what is asked for fits alone."""
        while asked and len(self.scheduler.running) + len(self.scheduler.waiting) < self.cfg.max_num_seqs:
            ids, sp = asked[0]
            pages = (len(ids) - 1) // self.cfg.block_size          # all in front of the last token
            prefix = None
            if pages:
                if self.has_work() and (self._no_room_for_prefix(pages)
                                        or not self.scheduler.can_ever_fit(self._most_positions(len(ids), sp), pages, pinned=pages)):
                    return
                prefix = self.add_prefix(ids[:pages * self.cfg.block_size])
            asked.popleft()
            try:
                for _ in range(n):
                    seqs.append(self.add_request(ids, sp, prefix=prefix))
                    seqs[-1].arrival_time = arrival
            finally:
                if prefix is not None:                             # (held by the requests that begin with it)
                    self.release_prefix(prefix)

    def generate(self, prompts, params=None, decode_text: bool = True, n: int = 1) -> list:
        """``n`` answers to every prompt, one behind another in the result; with more than one, the answers to a prompt share its pages where the
        model allows it (``add_prefix``), and steps read them once for all of a prompt's answers where that pays, for up to
        ``SHARED_GROUPS`` prompts at a time (with more, every answer reads them by itself).  A prompt's pages are computed and held once its answers' turn comes: prompts that do not fit the cache side by
        side wait for those in front.  What cannot be run at all is refused with ValueError before anything is added."""
        if not isinstance(params, list):
            params = [params or SamplingParams()] * len(prompts)
        if len(params) != len(prompts):
            raise ValueError("one SamplingParams per prompt")
        if n < 1:
            raise ValueError(f"n must be at least 1, got {n}")
        arrival = time.perf_counter()
        asked = deque(self._checked(p, sp) for p, sp in zip(prompts, params))
        for ids, sp in asked:
            self._refuse_what_never_fits(len(ids), sp)
        seqs: list = []
        if n == 1 or not self.can_share:
            seqs = [self.add_request(ids, sp) for ids, sp in asked for _ in range(n)]
            asked.clear()
        while asked or self.has_work():
            self._add_answers(asked, n, seqs, arrival)
            self.step()
        outs = []
        for s in seqs:
            text = None
            if decode_text and self.tokenizer is not None:
                text = self.tokenizer.decode(s.output_ids, skip_special_tokens=True)
            first = None if s.first_token_time is None else s.first_token_time - s.arrival_time      # (a grammar may allow no token at all)
            outs.append(RequestOutput(s.seq_id, s.prompt_len, s.output_ids, text, first, s.finish_time - s.arrival_time,
                                      s.logprobs if s.params.logprobs else None))
        return outs
