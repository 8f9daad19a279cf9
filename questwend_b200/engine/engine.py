"""The engine: a model, its cache, and the one step function.

``step`` takes a batch of sequences, each with its next tokens (a whole prompt, or
one token), runs exactly those tokens as one packed batch against the cache that
earlier steps left, and returns the logits at the places asked for.  There is no
padding anywhere: sequences of unequal length are packed end to end, and the
kernels take each sequence's own start and length.

The reference's counterpart is ``Runtime::decode`` for one sequence
(core/runtime.cpp:3020-3203 for a prompt, :1768-1829 for one token), which
returns the last position's logits only (core/runtime.h:52-54).
"""
from __future__ import annotations

import contextlib
from dataclasses import dataclass, field

import numpy as np
import torch

from .. import models  # noqa: F401  (registers the architectures)
from ..cache.manager import CacheManager, pages_for
from ..config.base import ModelConfig
from ..config.registry import get_architecture, load_config
from ..kernels import build as kernel_build
from ..kernels import ops
from ..kernels.ops import PAGE_SIZE, fill_int32
from ..parts.base import KVSpec, Runtime, StepContext
from ..parts.linear import require_true_fp32
from ..weights.loader import load_tensors
from ..weights.random_init import random_tensors
from .model import Model

DTYPES = {"bfloat16": torch.bfloat16, "bf16": torch.bfloat16, "float32": torch.float32, "fp32": torch.float32,
          torch.bfloat16: torch.bfloat16, torch.float32: torch.float32}


class EngineError(RuntimeError):
    pass


@dataclass
class StepEntry:
    """One sequence's part of a step: its slot, its next tokens, and the places among
    these tokens (0-based) whose logits are wanted."""
    slot: int
    tokens: list
    want: list = field(default_factory=list)


def _require_cuda(device: torch.device) -> None:
    if device.type != "cuda":
        raise EngineError(f"the engine runs on a CUDA device only, got '{device}' (there is no CPU path)")
    if not torch.cuda.is_available():
        raise EngineError("no CUDA device is available; the engine has no CPU path")
    major, minor = torch.cuda.get_device_capability(device)
    if (major, minor) != (10, 0):
        raise EngineError(f"the kernels are built for sm_100a (B200); this device is sm_{major}{minor}")


def build_step_context(cache: CacheManager, entries: list, vocab_size: int, device) -> tuple[StepContext, torch.Tensor]:
    """Pack one step's entries for the device: reserves cache pages for the new tokens (or raises and
    changes nothing), and returns the context and the packed rows whose logits are wanted."""
    if not entries:
        raise EngineError("a step needs at least one sequence")
    slots = [e.slot for e in entries]
    if len(set(slots)) != len(slots):
        raise EngineError(f"a slot appears twice in one step: {slots}")
    B = len(entries)
    if B > ops.STEP_TABLES_MAX_SEQS:
        raise EngineError(f"a step takes up to {ops.STEP_TABLES_MAX_SEQS} sequences, not {B}")
    n_new = []
    for e in entries:
        if len(e.tokens) == 0:
            raise EngineError(f"slot {e.slot}: a step must bring at least one token for each sequence")
        n_new.append(len(e.tokens))
    T = sum(n_new)
    pos0 = [cache.length(s) for s in slots]

    ids, want = np.empty(T, dtype=np.int32), []
    t = 0
    for b, e in enumerate(entries):
        n = n_new[b]
        if not fill_int32(ids[t:t + n], e.tokens):
            try:
                ids[t:t + n] = e.tokens
            except (TypeError, ValueError, OverflowError):
                raise EngineError(f"slot {e.slot}: token ids must be integers") from None
        for i in e.want:
            if not 0 <= i < n:
                raise EngineError(f"slot {e.slot}: wanted place {i} is outside this step's {n} tokens")
            want.append(t + i)
        t += n
    if T and (ids.min() < 0 or ids.max() >= vocab_size):
        bad = int(ids[(ids < 0) | (ids >= vocab_size)][0])
        raise EngineError(f"token id {bad} is outside the vocabulary of {vocab_size}")
    slen = [p + n for p, n in zip(pos0, n_new)]
    cache.reserve(dict(zip(slots, slen)))     # after every check: a refused step holds nothing
    # What only the host knows goes to the device in one copy: the tokens, each sequence's length, count and slot, the places wanted,
    # and for each cache group where each sequence's pages begin and the pages, one sequence after the other.  Everything else is made
    # of it there (``ops.step_tables``: a launch a group).
    groups = cache.n_groups()
    rest, sizes = [*pos0, *n_new, *slots, *want], [T, B, B, B, len(want)]
    for gid in range(max(1, groups)):
        lists = cache.page_lists(gid, slots) if groups else [()] * B
        starts = [0]
        for pages in lists:
            starts.append(starts[-1] + len(pages))
        rest += starts
        for pages in lists:
            rest += pages
        sizes += [B + 1, starts[-1]]
    buf = np.empty(T + len(rest), dtype=np.int32)
    buf[:T] = ids
    if not fill_int32(buf[T:], rest):
        buf[T:] = rest
    dev = torch.from_numpy(buf).to(device)
    parts = dev.split(sizes)
    width = cache.table_width if groups else 0
    tables, first = {}, None
    with contextlib.nullcontext() if dev.get_device() == torch.cuda.current_device() else torch.cuda.device(dev.device):
        for gid in range(max(1, groups)):
            of_tokens = first is None or cache.group_spec(gid).bits == 4
            made = ops.step_tables(parts[6 + 2 * gid], parts[5 + 2 * gid], parts[1], parts[2], T, width, tokens=of_tokens)
            first = first or made
            if groups:
                tables[gid] = made
    ctx = StepContext(n_tokens=T, n_seqs=B, token_ids=parts[0], tok_seq=first.tok_seq, tok_pos=first.tok_pos,
                      cu_seqlens=first.cu_seqlens, pos0=parts[1], seq_len=first.seq_len, slots=parts[3],
                      max_new=max(n_new), min_new=min(n_new), max_len=max(slen), single_token=all(n == 1 for n in n_new),
                      page_tables={gid: t.page_table for gid, t in tables.items()}, host_slots=slots,
                      all_start=all(p == 0 for p in pos0), tables=tables)
    return ctx, parts[4]


def require_cache_bits(plan, cache_bits: int) -> None:
    """Refuse a cache in fewer bits that a mixer of this plan does not keep, before a weight is read."""
    if cache_bits == 0:
        return
    if cache_bits != 4:
        raise EngineError(f"cache_bits: keys and values are cached in the engine's dtype (0) or in 4 bits (4), not in {cache_bits}")
    try:
        model = Model(plan, Runtime(torch.device("cpu"), torch.bfloat16, cache_bits))
    except ValueError as e:
        raise EngineError(f"cache_bits=4: {e}") from None
    found = 0
    for run, (kv, _, _) in zip(plan.schedule, model.cache_units()):
        for spec in () if kv is None else (kv,) if isinstance(kv, KVSpec) else kv:
            found += 1
            if spec.bits != cache_bits:
                raise EngineError(f"cache_bits=4: layer {run.layer}'s mixer '{plan.layers[run.layer].mixer.kind}' keeps its cache in the "
                                  f"engine's dtype only")
    if not found:
        raise EngineError("cache_bits=4: this model caches no keys and values")


class Engine:
    """Build with ``Engine.from_folder`` or ``Engine.from_config``.

    max_tokens   the most tokens live sequences hold together (each rounded up to pages of 64)
    max_seq_len  the longest single sequence (default: max_tokens, capped by the model's trained length)
    max_batch    the most sequences alive at once (default: as many as could each hold one page, up to 256)
    cache_bits   4: keys and values are cached in 4 bits, a step for 32 of them (3.6 times as many tokens in the same memory as in
                 bfloat16; the cache's numbers are then off by 2 % of a row's size, so logits differ from those of a cache in the
                 engine's dtype); grouped-query attention only.  0: in the engine's dtype
    """

    def __init__(self, config: ModelConfig, weights: dict, dtype: torch.dtype, device: torch.device,
                 max_tokens: int, max_seq_len: int | None = None, max_batch: int | None = None, cache_bits: int = 0):
        self.config = config
        self.dtype = dtype
        self.cache_bits = cache_bits
        self.device = device
        if dtype == torch.float32:
            require_true_fp32()
        arch = get_architecture(config.architecture)
        self.plan = arch.plan(config)
        require_cache_bits(self.plan, cache_bits)
        self.runtime = Runtime(device, dtype, cache_bits)
        self.model = Model(self.plan, self.runtime)
        kernel_build.compile_modules(["step_tables", *self.model.kernel_modules()])
        self.model.bind(weights)
        self.vocab_size = self.plan.vocab_size
        if max_seq_len is None:
            max_seq_len = max_tokens
            if self.plan.max_position:
                max_seq_len = min(max_seq_len, self.plan.max_position)
        if self.plan.position_limit and max_seq_len > self.plan.position_limit:
            raise EngineError(f"max_seq_len {max_seq_len}: this model has {self.plan.position_limit} positions")
        max_seq_len = min(max_seq_len, pages_for(max_tokens) * PAGE_SIZE)
        if max_batch is None:
            max_batch = max(1, min(256, pages_for(max_tokens)))
        self.max_batch = max_batch
        self.cache = CacheManager(self.model.cache_units(), max_tokens, max_batch, max_seq_len, dtype, device)
        self.unit_caches = [self.cache.unit_cache(i) for i in range(len(self.model.schedule))]
        self.steps_run = 0
        self._runners: dict = {}

    # ------------------------------------------------------------------ construction
    @classmethod
    def from_folder(cls, model_dir: str, dtype="bfloat16", device="cuda:0", **kw) -> "Engine":
        device = torch.device(device)
        _require_cuda(device)
        dtype = DTYPES[dtype]
        config = load_config(model_dir)
        plan = get_architecture(config.architecture).plan(config)
        require_cache_bits(plan, kw.get("cache_bits", 0))
        weights = load_tensors(model_dir, plan.manifest(), dtype, device)
        return cls(config, weights, dtype, device, **kw)

    @classmethod
    def from_config(cls, config: ModelConfig, seed: int, dtype="bfloat16", device="cuda:0", **kw) -> "Engine":
        """Random weights drawn on the device (the values differ from a folder written with the same seed)."""
        device = torch.device(device)
        _require_cuda(device)
        dtype = DTYPES[dtype]
        plan = get_architecture(config.architecture).plan(config)
        require_cache_bits(plan, kw.get("cache_bits", 0))
        weights = random_tensors(plan.manifest(), seed, dtype, device=device, vector_dtype=torch.float32)
        return cls(config, weights, dtype, device, **kw)

    # ------------------------------------------------------------------ sequences
    def open_sequences(self, count: int) -> list[int]:
        return self.cache.open(count)

    def close_sequences(self, slots) -> None:
        self.cache.close(slots)

    # ------------------------------------------------------------------ the step
    def build_context(self, entries: list[StepEntry]) -> tuple[StepContext, torch.Tensor]:
        return build_step_context(self.cache, entries, self.vocab_size, self.device)

    @torch.no_grad()
    def step(self, entries: list[StepEntry]) -> torch.Tensor:
        """Run the entries' tokens; returns float32 logits [wanted, vocab] on the device, in the
        order of the entries and of each entry's ``want``."""
        with torch.cuda.device(self.device):
            ctx, want_rows = self.build_context(entries)
            logits = self.model.forward(ctx, self.unit_caches, want_rows)
            self.check_kernels()
        for e in entries:
            self.cache.advance(e.slot, len(e.tokens))
        self.steps_run += 1
        return logits

    def check_kernels(self) -> None:
        """Raise if a kernel with bounded waits (the TMA-fed products, the tcgen05 attention, in both engines the recurrences in
        chunks) gave one up since the last check: its result is then not valid.  Reads one int from the device, so it waits for the
        work queued so far, if such a kernel was launched at all."""
        with torch.cuda.device(self.device):
            ops.gemm_tc_check(self.device)

    def decode_runner(self, batch: int, sampling, use_graph: bool = True, logprobs: int | None = None):
        """The fixed buffers and CUDA graphs for decode steps of ``batch`` sequences (made once, kept).  The sampling
        options without the seed key it: the seed lives on the device and is given with ``bind``.  ``logprobs``: also the sampled
        tokens' log probabilities, with so many alternatives each."""
        import dataclasses
        from .decode import DecodeRunner
        sampling = dataclasses.replace(sampling, seed=0)
        key = (batch, sampling, use_graph, logprobs)
        runner = self._runners.get(key)
        if runner is None:
            if len(self._runners) >= 16:             # graphs hold memory: drop the oldest
                self._runners.pop(next(iter(self._runners)))
            runner = self._runners[key] = DecodeRunner(self, batch, sampling, use_graph, logprobs)
        return runner

    # ------------------------------------------------------------------ facts
    def describe(self) -> dict:
        n_params = sum(int(np.prod(t.shape)) for t in self.model.tensors() if not (t.optional or t.ignored))
        return {"architecture": self.config.architecture, "dtype": str(self.dtype).replace("torch.", ""),
                "parameters": n_params, "cache_bits": self.cache_bits or 8 * torch.empty((), dtype=self.dtype).element_size(),
                "cache_bytes": self.cache.bytes_held(),
                "max_tokens": self.cache.max_tokens, "max_seq_len": self.cache.max_seq_len,
                "max_batch": self.max_batch, "page_size": PAGE_SIZE, "layers": len(self.plan.layers),
                "schedule": len(self.plan.schedule), "cache_groups": self.cache.n_groups()}
