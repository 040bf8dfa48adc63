"""Choosing the next token of every request of a step, on the device.

Greedy rows use the argmax kernel; rows with a temperature use the sampling kernel (temperature,
top-k, top-p; a counter-based uniform draw keyed by the request's seed and the index of the draw, so
a request's tokens do not depend on what else is in the batch or on being recomputed after a
preemption).  Penalties, biases, banned ids and grammars are applied to the logits first, all of a step's in one
kernel (``ops.logit_rules``) whose inputs travel in one copy.

Reference parity: ``src/scheduler/continuous_batch_engine.cpp:237,259-305`` (greedy on the last row of
each request) and ``demo/qwen3_infer.cpp:229-423`` (the sampler of the single-stream demo).
"""
from __future__ import annotations

import numpy as np
import torch

from .. import ops
from .params import SamplingParams


class Sampler:
    """Sampling options live in small device tables, one entry per distinct set of options, written once when a
    request with new options first samples.  A step then ships only one int64 pair per row - (table entry, draw
    counter) - in a single copy from pinned memory."""

    def __init__(self, device, table_entries: int = 1024, max_rows: int = 256):
        self.device = torch.device(device)
        self.table_entries = table_entries
        self._entry_of: dict = {}             # (temperature, top_k, top_p, seed) -> entry, in order of last use
        self._tables = None
        self._staging: list = []              # pinned buffers for the per-step pairs, used in turn
        self._copied: list = []
        self._turn = 0
        self._max_rows = max_rows

    # ---- option tables -------------------------------------------------------------------------------------
    def _ensure_tables(self) -> None:
        if self._tables is None:
            n, dev = self.table_entries, self.device
            self._tables = (torch.zeros(n, dtype=torch.float32, device=dev), torch.zeros(n, dtype=torch.int32, device=dev),
                            torch.zeros(n, dtype=torch.float32, device=dev), torch.zeros(n, dtype=torch.int64, device=dev))

    def _entry(self, p: SamplingParams) -> int:
        key = (0.0 if p.greedy else float(p.temperature), int(p.top_k), float(p.top_p), _as_i64(p.seed))
        entry = self._entry_of.pop(key, None)
        if entry is None:
            if len(self._entry_of) < self.table_entries:
                entry = len(self._entry_of)
            else:                              # the table is full: the entry unused for longest is overwritten
                oldest = next(iter(self._entry_of))
                entry = self._entry_of.pop(oldest)
            temperature, top_k, top_p, seeds = self._tables
            temperature[entry], top_k[entry], top_p[entry], seeds[entry] = key
        self._entry_of[key] = entry            # most recently used last
        return entry

    def _pairs_to_device(self, pairs: list) -> torch.Tensor:
        n = len(pairs)
        if not self._staging or self._staging[0].shape[0] < n:
            self._max_rows = max(self._max_rows, n)
            self._staging = [torch.empty((self._max_rows, 2), dtype=torch.int64).pin_memory() for _ in range(4)]
            self._copied = [None] * 4
        i = self._turn
        self._turn = (self._turn + 1) % len(self._staging)
        if self._copied[i] is not None:
            self._copied[i].synchronize()      # the copy that last used this buffer has run
        host = self._staging[i][:n]
        host.copy_(torch.tensor(pairs, dtype=torch.int64))
        dev = host.to(self.device, non_blocking=True)
        self._copied[i] = torch.cuda.Event()
        self._copied[i].record()
        return dev

    def sample(self, logits: torch.Tensor, params: list, draw_index: list, history: list | None = None,
               prompt_lens: list | None = None, allowed: list | None = None) -> list:
        """logits float32 [n, V]; params[i] SamplingParams; draw_index[i] how many tokens request i has
        drawn so far; history[i] the tokens that penalties and grammars look at (ids, a list or an int32 array), its first
        prompt_lens[i] (default: none) the prompt; allowed[i] what request i's grammar allows (``SamplingParams.token_mask``;
        asked for here if ``allowed`` is not given).  Returns n token ids; -1 where the rules leave no token."""
        out = self.sample_device(logits, params, draw_index, history, prompt_lens, allowed)
        return [] if out is None else out.tolist()

    def _apply_rules(self, logits: torch.Tensor, params: list, history: list | None, prompt_lens: list | None,
                     allowed: list | None) -> torch.Tensor:
        """``logits`` after the rules of every row, in a new tensor."""
        n, V = logits.shape
        if n > 1 and logits.stride(0) < V:               # a row that several requests share
            logits = logits.contiguous()
        told = history is not None
        tokens = [np.asarray(history[i], dtype=np.int32) if told and p.needs_history else np.empty(0, np.int32)
                  for i, p in enumerate(params)]
        prompts = [min(int(prompt_lens[i]), tokens[i].size) if prompt_lens is not None else 0 for i in range(n)]
        biases = []
        for p in params:
            row = dict(p.logit_bias)
            row.update((t, float("-inf")) for t in p.banned_tokens)
            biases.append({t: v for t, v in row.items() if 0 <= t < V})     # ids that are none may be beyond 32 bits
        if allowed is None:
            allowed = [p.token_mask(tokens[i][prompts[i]:].tolist(), V) for i, p in enumerate(params)]
        masks = [m for m in allowed if m is not None]
        ends = np.cumsum([m is not None for m in allowed])
        mask_row = [int(end) - 1 if m is not None else -1 for m, end in zip(allowed, ends)]
        f32 = lambda v: np.asarray(v, dtype=np.float32).view(np.int32)  # noqa: E731
        off = lambda v: np.concatenate([[0], np.cumsum(v)]).astype(np.int32)  # noqa: E731
        with_history = [p.needs_history and told for p in params]
        parts = [off([t.size for t in tokens]), np.asarray(prompts, np.int32),
                 f32([p.repetition_penalty if h else 1.0 for p, h in zip(params, with_history)]),
                 f32([p.frequency_penalty if h else 0.0 for p, h in zip(params, with_history)]),
                 f32([p.presence_penalty if h and p.presence_penalty > 0.0 else 0.0 for p, h in zip(params, with_history)]),
                 np.concatenate(tokens), off([len(b) for b in biases]), np.asarray([t for b in biases for t in b], np.int32),
                 f32([v for b in biases for v in b.values()]), np.asarray(mask_row, np.int32),
                 np.concatenate(masks) if masks else np.empty(0, np.int32)]
        host = torch.from_numpy(np.concatenate(parts))
        if self.device.type == "cuda":
            host = host.pin_memory()
        (history_off, prompt_len, repetition, frequency, presence, flat, bias_off, bias_tokens, bias_values, rows,
         mask) = host.to(self.device, non_blocking=True).split([p.size for p in parts])
        as_f32 = lambda t: t.view(torch.float32)  # noqa: E731
        kw = {}
        if bias_tokens.numel():
            kw.update(bias_off=bias_off, bias_tokens=bias_tokens, bias_values=as_f32(bias_values))
        if masks:
            kw.update(mask=mask.view(len(masks), -1), mask_row=rows)
        return ops.logit_rules(logits, flat, history_off, prompt_len, as_f32(repetition), as_f32(frequency), as_f32(presence), **kw)

    def sample_device(self, logits: torch.Tensor, params: list, draw_index: list, history: list | None = None,
                      prompt_lens: list | None = None, allowed: list | None = None):
        """The same, but the token ids stay on the device (int32 [n], or None for no rows): the caller reads them
        when it needs them, and the next step can take them as its input without a round trip."""
        n = logits.shape[0]
        if n == 0:
            return None
        if any(p.edits_logits for p in params):
            logits = self._apply_rules(logits, params, history, prompt_lens, allowed)
        if all(p.greedy for p in params):
            return ops.argmax(logits)
        self._ensure_tables()
        if n > self.table_entries:
            raise ValueError(f"{n} rows in one step, the sampler's option tables hold {self.table_entries} entries")
        pairs = [[self._entry(p), int(c)] for p, c in zip(params, draw_index)]
        temperature, top_k, top_p, seeds = self._tables
        return ops.sample_entries(logits, temperature, top_k, top_p, seeds, self._pairs_to_device(pairs))


def _as_i64(v: int) -> int:
    v &= (1 << 64) - 1
    return v - (1 << 64) if v >= (1 << 63) else v
