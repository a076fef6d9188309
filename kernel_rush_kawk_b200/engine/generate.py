"""The generation loop above the step function.

A batch of prompts of unequal lengths starts together: all prompts in one step,
then one token per live sequence per step. A sequence ends when it has produced
``max_new_tokens`` tokens or one of its stop tokens; it then gives its slot and
pages back and the batch goes on without it. ``run_requests`` runs as many
batches one after another as the requests need, each batch as large as the
cache allows.

The reference's loop (``GraphPlan.run``, engine/engine.py:438-469 of
willzeng274/kernel-rush-kawk) serves equal-length prompts, never stops on a
token (EOS is an ordinary id: AGENTS.md:19-21) and yields exactly
``max_new_tokens`` lists. With no stop tokens this loop yields the same.

Like the reference's, which keeps up to three decode replays queued behind a ring
of pinned token buffers with one event each (engine.py:81-83,458-469), the loop
runs ahead of its consumer where the step function offers it (``open_decode_run``):
each single-token step takes its tokens on the device from the selection kernel of
the step before, so up to ``RUN_AHEAD`` steps are queued while the host reads an
earlier step's tokens. When a read shows that a sequence has stopped, nothing more
is queued; the steps already queued still ran that sequence (into pages it gives
back afterwards) and their tokens for it are dropped. The batch then goes on,
smaller, from the host's tokens.

With ``share_prefix`` the prompts stand in the order of their tokens, and neighbours that begin with the same whole
pages form a group (``shared_prefixes``): the first of them runs those pages' tokens, the others' sequences are
forked from it, and all bring the rest of their prompts in the next step.
"""

from __future__ import annotations

import time
from dataclasses import dataclass, field

from ..cache.eviction import KeyEviction
from ..cache.store import PAGE
from ..sampling.sampler import SamplingParams
from .step import StepEntry


@dataclass
class Sequence:
    request: int
    prompt: list
    adapter: int = -1
    slot: int = -1
    produced: list = field(default_factory=list)
    finished: bool = False
    reason: str = ""


@dataclass
class GenerationStats:
    """What one batch of ``run_batch`` took, by the host's clock. The reference logs
    the like per plan (``GraphPlan.stats`` and its log lines, engine/engine.py:87,206,378)."""
    sequences: int = 0
    prompt_tokens: int = 0
    shared_tokens: int = 0         # of these, the ones that did not run because another prompt's had
    prefill_ms: float = 0.0        # from the call to the first tokens on the host
    decode_steps: int = 0          # single-token steps whose tokens were read
    decode_ms: float = 0.0         # from the first tokens to the last ones
    new_tokens: int = 0

    @property
    def decode_ms_per_step(self) -> float:
        return self.decode_ms / self.decode_steps if self.decode_steps else 0.0

    @property
    def decode_tokens_per_s(self) -> float:
        decoded = self.new_tokens - self.sequences
        return decoded * 1000.0 / self.decode_ms if self.decode_ms > 0 and decoded > 0 else 0.0

    @property
    def prefill_tokens_per_s(self) -> float:
        return (self.prompt_tokens - self.shared_tokens) * 1000.0 / self.prefill_ms if self.prefill_ms > 0 else 0.0

    def line(self) -> str:
        shared = f" ({self.shared_tokens} shared)" if self.shared_tokens else ""
        return (f"{self.sequences} sequences, {self.prompt_tokens} prompt tokens{shared} in {self.prefill_ms:.1f} ms "
                f"({self.prefill_tokens_per_s:.0f} tokens/s); {self.decode_steps} decode steps at "
                f"{self.decode_ms_per_step:.3f} ms ({self.decode_tokens_per_s:.0f} tokens/s)")


def rows_held(prompt_len: int, max_new_tokens: int, eviction: KeyEviction | None = None, pass_tokens: int | None = None) -> int:
    """The most rows of the cache that a sequence comes to hold: the last generated token is never fed back. Where keys are evicted, it holds fewer than
    ``keep + every`` before a step, and what the step brings beside them: a piece of its prompt, of ``pass_tokens`` at most, or one token."""
    rows = prompt_len + max(max_new_tokens - 1, 0)
    if eviction is None:
        return rows
    full = eviction.keep + eviction.every
    return min(rows, max(full, prompt_len if pass_tokens is None else min(prompt_len, full - 1 + pass_tokens)))


def pages_needed(prompt_len: int, max_new_tokens: int, eviction: KeyEviction | None = None, pass_tokens: int | None = None) -> int:
    """Pages that these rows take."""
    return -(-rows_held(prompt_len, max_new_tokens, eviction, pass_tokens) // PAGE)


def shared_prefixes(prompts: list, adapters=None) -> list:
    """Groups of prompts that begin alike, and run with the same adapter (``adapters``: theirs, -1 for none), whose keys are others: (request indices, tokens shared) with the shared tokens whole pages, at least one token of
    every prompt behind them, 0 for a prompt alone. Neighbours in the order of the prompts' tokens join a group while the pages that it
    saves, (members - 1) * shared pages, do not get fewer."""
    of = adapters or [-1] * len(prompts)
    order = sorted(range(len(prompts)), key=lambda i: (of[i], prompts[i]))
    groups: list = []
    for i in order:
        p = prompts[i]
        if groups:
            members, shared = groups[-1]
            other = prompts[members[0]]
            most = min(len(p) - 1, shared if len(members) > 1 else len(other) - 1)
            n = 0
            if of[i] != of[members[0]]:
                most = 0
            while n < most and p[n] == other[n]:
                n += 1
            n -= n % PAGE
            if n > 0 and len(members) * n >= (len(members) - 1) * shared:
                groups[-1] = (members + [i], n)
                continue
        groups.append(([i], 0))
    return groups


def shared_pages(prompts: list, max_new_tokens: int, adapters=None) -> int:
    """Pages that a batch of prompts comes to hold which share what they begin with: a group's shared ones count once."""
    pages = sum(pages_needed(len(p), max_new_tokens) for p in prompts)
    return pages - sum((len(members) - 1) * (shared // PAGE) for members, shared in shared_prefixes(prompts, adapters))


def split_into_batches(prompt_lens: list, max_new_tokens: int, max_slots: int, max_pages: int, eviction: KeyEviction | None = None,
                       pass_tokens: int | None = None, prompts: list | None = None, adapters=None) -> list:
    """Consecutive requests are grouped while slots and pages last. Returns lists of
    request indices. A request that cannot fit even alone raises ValueError. ``prompts``: theirs, where a batch shares what they begin with."""
    needs = [pages_needed(n, max_new_tokens, eviction, pass_tokens) for n in prompt_lens]
    for i, need in enumerate(needs):
        if need > max_pages:
            raise ValueError(f"request {i} needs {need * PAGE} cached tokens; the cache holds {max_pages * PAGE}")
    batches, first, n = [], 0, len(needs)
    while first < n:
        most = min(n - first, max(max_slots, 1))
        size, pages = 1, needs[first]
        while size < most and pages + needs[first + size] <= max_pages:
            pages += needs[first + size]
            size += 1
        if prompts is not None and size < most:  # more fit where pages are shared: all that there are slots for, or as many as halving finds
            low, high = size, most + 1
            while high - low > 1:
                middle = most if high > most else (low + high) // 2
                fits = shared_pages(prompts[first:first + middle], max_new_tokens, adapters and adapters[first:first + middle]) <= max_pages
                low, high = (middle, high) if fits else (low, middle)
            size = low
        batches.append(list(range(first, first + size)))
        first += size
    return batches


class GenerationLoop:
    RUN_AHEAD = 3  # single-token steps queued on the device while the host reads an earlier one

    def __init__(self, stepper, cache, sampler):
        self.stepper = stepper
        self.cache = cache
        self.sampler = sampler
        self.steps = 0
        self.stats = GenerationStats()  # of the last batch

    def run_batch(self, prompts: list, max_new_tokens: int, sampling: SamplingParams = SamplingParams(),
                  stop_token_ids=(), first_request: int = 0, share_prefix: bool = False, adapters=None):
        """Generator: yields, per step, a list with one entry per prompt: the new token
        id, or None for a sequence that ended at an earlier step. ``adapters``: the low-rank adapter of each prompt (-1: none)."""
        if max_new_tokens < 1 or not prompts:
            return
        for i, p in enumerate(prompts):
            if len(p) == 0:
                raise ValueError(f"prompt {i} is empty")
        stops = frozenset(int(t) for t in stop_token_ids)
        seqs = [Sequence(first_request + i, list(p), -1 if adapters is None else adapters[i]) for i, p in enumerate(prompts)]
        stats = self.stats = GenerationStats(len(seqs), sum(len(p) for p in prompts))
        t_begin = time.perf_counter()
        t_first = None

        def take(live, tokens):
            """Book one step's tokens; returns (what to yield, who goes on)."""
            out = [None] * len(seqs)
            still = []
            for s, tok in zip(live, tokens):
                if s.finished:  # stopped at a step read earlier: this one ran ahead of that news
                    continue
                s.produced.append(tok)
                stats.new_tokens += 1
                out[s.request - first_request] = tok
                if tok in stops:
                    s.finished, s.reason = True, "stop"
                elif len(s.produced) >= max_new_tokens:
                    s.finished, s.reason = True, "length"
                if not s.finished:
                    still.append(s)
            self.steps += 1
            return out, still

        def release(group):
            for s in group:
                if s.finished and s.slot >= 0:
                    self.cache.free(s.slot)
                    s.slot = -1

        if share_prefix and not self.cache.can_share():
            raise ValueError("prompts cannot share their beginnings in this engine: a layer keeps a window of keys, or keys are evicted")
        try:
            if share_prefix:
                live, begun, stats.shared_tokens = self._start_shared(seqs)
            else:
                for s in seqs:
                    s.slot = self.cache.alloc(s.adapter)
                live, begun = list(seqs), [0] * len(seqs)
            logits = self.stepper.step([StepEntry(s.slot, s.prompt[n:], [len(s.prompt) - 1 - n]) for s, n in zip(live, begun)])
            tokens = self.sampler.select(logits, sampling, [s.request for s in live], 0)
            t_first = time.perf_counter()
            stats.prefill_ms = (t_first - t_begin) * 1e3
            out, still = take(live, tokens)
            release(live)
            live = still
            yield out
            open_run = getattr(self.stepper, "open_decode_run", None)
            while live:
                step = len(live[0].produced)  # every live sequence has produced this many tokens
                requests = [s.request for s in live]
                last = [s.produced[-1] for s in live]
                run = open_run([s.slot for s in live], last, sampling, requests, step, self.RUN_AHEAD) if open_run else None
                if run is None:  # one step at a time, tokens through the host
                    logits = self.stepper.step([StepEntry(s.slot, [t], [0]) for s, t in zip(live, last)])
                    tokens = self.sampler.select(logits, sampling, requests, step)
                    stats.decode_steps += 1
                    stats.decode_ms = (time.perf_counter() - t_first) * 1e3
                    out, still = take(live, tokens)
                    release(live)
                    live = still
                    yield out
                    continue
                # the last token of a sequence is never fed back: max_new_tokens - step steps remain
                to_launch = max_new_tokens - step
                group, stopping = live, False
                while True:
                    while to_launch > 0 and not stopping and run.in_flight < self.RUN_AHEAD:
                        run.launch()
                        to_launch -= 1
                    if run.in_flight == 0:
                        break
                    tokens = run.collect()
                    stats.decode_steps += 1
                    stats.decode_ms = (time.perf_counter() - t_first) * 1e3
                    out, still = take(group, tokens)
                    stopping = stopping or len(still) < len(live)
                    live = still
                    if any(t is not None for t in out):
                        yield out
                release(group)
        finally:
            for s in seqs:
                if s.slot >= 0:
                    self.cache.free(s.slot)
                    s.slot = -1

    def _start_shared(self, seqs: list) -> tuple[list, list, int]:
        """Run what the prompts share, once; (the sequences in the order of their groups, the tokens that each has had, how many of these in all did
        not run again)."""
        order, begun, first = [], [], []
        groups = [([seqs[i] for i in members], shared) for members, shared in shared_prefixes([s.prompt for s in seqs], [s.adapter for s in seqs])]
        for members, shared in groups:
            members[0].slot = self.cache.alloc(members[0].adapter)
            if shared:
                first.append(StepEntry(members[0].slot, members[0].prompt[:shared], []))
        if first:
            self.stepper.step(first)
        for members, shared in groups:
            for s in members[1:]:
                s.slot = self.cache.fork(members[0].slot, shared)
            order += members
            begun += [shared] * len(members)
        return order, begun, sum((len(members) - 1) * shared for members, shared in groups)

    def run_requests(self, prompts: list, max_new_tokens: int, sampling: SamplingParams = SamplingParams(),
                     stop_token_ids=(), max_batch: int | None = None, share_prefix: bool = False, adapters=None) -> list:
        """Run every request, batch after batch; returns each request's generated tokens."""
        max_slots = min(self.cache.max_slots, max_batch or self.cache.max_slots)
        batches = split_into_batches([len(p) for p in prompts], max_new_tokens, max_slots, self.cache.n_pages, self.cache.eviction,
                                     getattr(self.stepper, "max_step_rows", None), prompts if share_prefix else None, adapters)
        results: list = [None] * len(prompts)
        for batch in batches:
            outs = [[] for _ in batch]
            for step_out in self.run_batch([prompts[i] for i in batch], max_new_tokens, sampling, stop_token_ids,
                                           first_request=batch[0], share_prefix=share_prefix,
                                           adapters=adapters and [adapters[i] for i in batch]):
                for j, tok in enumerate(step_out):
                    if tok is not None:
                        outs[j].append(tok)
            for j, i in enumerate(batch):
                results[i] = outs[j]
        return results
