"""The generation loop above the step function.

Per batch: all prompts in one step, a token sampled for each sequence from the logits of its
prompt's last place, then one token per live sequence per step. `max_tokens` counts the token
sampled from the prompt's logits, so at least one token is always produced; a stop token is kept
in the output and counted, and ends its sequence; the last sampled token is not fed back
(model_f32.go:604-669). A prompt longer than the engine can hold keeps its tail
(model_f32.go:598-602). Sequences of a batch end independently; requests beyond what fits at once
run as further batches on the slots the earlier ones gave back.

Prompts that begin alike can share what they begin with (`share_prefix`, and `n` continuations of each prompt): the common run of
tokens goes through the model once, its sequence is forked for the others, and later steps read its pages once for all. The sampled
tokens are those that the requests would give alone, but for rounding.

The loop's decisions (who is live, who stops and why, how requests are split into batches) are
plain Python over token ids, so they can be tested with a scripted step function.
"""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import Callable, Sequence as Seq

import numpy as np
import torch

from ..cache.needs import PAGE
from ..sampling.sampler import SamplingOptions


@dataclass
class GenerationResult:
    tokens: list[int]                 # sampled tokens, a final stop token included
    prompt_tokens: int
    finish_reason: str                # "stop" | "length" | "capacity" | "cancelled"
    prefill_ms: float = 0.0           # of the batch the request ran in
    decode_ms: float = 0.0

    @property
    def generated_tokens(self) -> int:
        return len(self.tokens)


def plan_batches(prompt_lens: Seq[int], max_tokens: int, max_seqs: int, page_capacity: int,
                 max_positions: int, n: int = 1) -> list[list[int]]:
    """Split request indices, in order, into batches that fit `max_seqs` slots and `page_capacity`
    cache pages when every request runs to its longest (prompt + max_tokens - 1 tokens held). With `n` > 1 requests n k to
    n k + n - 1 are one prompt: within a batch those behind the first need no pages for what they share."""
    batches, cur, cur_pages = [], [], 0
    for i, length in enumerate(prompt_lens):
        own, shared = request_pages(length, max_tokens, max_positions)
        if own + shared > page_capacity:
            held = min(max_positions, min(length, max_positions) + max_tokens - 1)
            raise ValueError(f"request {i} needs {own + shared} cache pages ({held} tokens); the cache has {page_capacity}")
        again = bool(cur) and i % n != 0
        if cur and (len(cur) >= max_seqs or cur_pages + own + (0 if again else shared) > page_capacity):
            batches.append(cur)
            cur, cur_pages, again = [], 0, False
        cur.append(i)
        cur_pages += own + (0 if again else shared)
    if cur:
        batches.append(cur)
    return batches


def request_pages(length: int, max_tokens: int, max_positions: int) -> tuple[int, int]:
    """Pages that a request needs when it runs to its longest: its own, and those that it shares with others of the same prompt (all
    of the prompt but its last token is shared, in whole pages)."""
    prompt = min(length, max_positions)
    held = min(max_positions, prompt + max_tokens - 1)
    shared = (prompt - 1) // PAGE
    return (max(held, 1) + PAGE - 1) // PAGE - shared, shared


def shared_runs(prompts: Seq[Seq[int]], alike: Seq | None = None) -> list[tuple[int, list[int], int, int]]:
    """What prompts begin with in common, as a tree: (depth, members, start, end) says that these prompts are the same up to `end`, and
    up to `start`, where their parent ends (0: they have none), with others too. Parents stand before their children. Every prompt keeps
    its last token for itself. With `alike`, only prompts with the same entry there are compared."""
    key = (lambda i: (alike[i], prompts[i])) if alike is not None else (lambda i: prompts[i])
    order = sorted(range(len(prompts)), key=key)
    arrays = [np.asarray(prompts[i], dtype=np.int64) for i in order]
    lcp = []
    for (i, a), (j, b) in zip(zip(order, arrays), zip(order[1:], arrays[1:])):
        n = min(len(a), len(b)) - 1
        same = a[:n] == b[:n]
        lcp.append(0 if alike is not None and alike[i] != alike[j] else n if same.all() else int(same.argmin()))
    runs, stack = [], [(0, len(order), 0, 0)]
    while stack:
        lo, hi, start, depth = stack.pop()
        if hi - lo < 2:
            continue
        m = min(lcp[lo:hi - 1])
        if m // PAGE > start // PAGE:          # a whole page more that is held once
            runs.append((depth, [order[k] for k in range(lo, hi)], start, m))
            start, depth = m, depth + 1
        at = lo
        for k in range(lo, hi):
            if k == hi - 1 or lcp[k] == m:
                stack.append((at, k + 1, start, depth))
                at = k + 1
    return sorted(runs, key=lambda r: r[0])


@dataclass
class _Live:
    request: int
    prompt: list[int]
    held: int                                     # tokens in the cache
    out: list[int] = field(default_factory=list)
    reason: str | None = None


class BatchState:
    """Who is live in a batch and what each has produced; no device code."""

    def __init__(self, requests: list[int], prompts: list[list[int]], max_tokens: int, stop_ids, max_positions: int):
        if max_tokens < 1:
            raise ValueError("max_tokens must be at least 1")
        self.max_tokens, self.stop_ids, self.max_positions = max_tokens, frozenset(stop_ids or ()), max_positions
        self.seqs = []
        for r, p in zip(requests, prompts):
            if len(p) == 0:
                raise ValueError(f"request {r} has an empty prompt")
            self.seqs.append(_Live(r, list(p[-max_positions:]), 0))

    def live(self) -> list[int]:
        return [i for i, s in enumerate(self.seqs) if s.reason is None]

    def accept(self, idx: list[int], fed: list[int], sampled: list[int]) -> list[int]:
        """Sequences `idx` were fed `fed[i]` tokens and sampled `sampled[i]`; returns those that just ended."""
        ended = []
        for i, n, t in zip(idx, fed, sampled):
            s = self.seqs[i]
            s.held += n
            s.out.append(int(t))
            if int(t) in self.stop_ids:
                s.reason = "stop"
            elif len(s.out) >= self.max_tokens:
                s.reason = "length"
            elif s.held + 1 > self.max_positions:
                s.reason = "capacity"
            if s.reason:
                ended.append(i)
        return ended

    def ends_by_count(self, i: int, fed: int) -> bool:
        """Whether sequence i ends with its next accepted token whatever that token is."""
        s = self.seqs[i]
        return len(s.out) + 1 >= self.max_tokens or s.held + fed + 1 > self.max_positions

    def cancel(self) -> list[int]:
        ended = self.live()
        for i in ended:
            self.seqs[i].reason = "cancelled"
        return ended


class Generator:
    """Runs requests through an Engine (or anything with open()/step()) and a Sampler."""

    def __init__(self, engine, sampler):
        self.engine, self.sampler = engine, sampler

    def _open(self, seqs: dict, n: int, state: BatchState, runs) -> list[int]:
        """Open a batch's sequences into `seqs`, the runs of tokens that they share run once, level by level of the tree, and their
        sequences forked for the members. Returns the prompt tokens that each holds already."""
        from .step import StepEntry
        done = [0] * n
        for depth in range(1 + max((r[0] for r in runs), default=-1)):
            level = [r for r in runs if r[0] == depth]
            for _, members, start, _ in level:
                if members[0] not in seqs:               # (a deeper run's members were forked with their parent's)
                    seqs[members[0]] = self.engine.open()
            self.engine.prompt_step([StepEntry(seqs[m[0]], state.seqs[m[0]].prompt[a:b]) for _, m, a, b in level])
            # a run's first member goes on with its sequence; the others, but for those that share a deeper run with one before, fork it
            deeper = {i: r[1][0] for r in runs if r[0] == depth + 1 for i in r[1]}
            for _, members, _, end in level:
                heads = [i for i in members[1:] if deeper.get(i, i) == i]
                seqs.update(zip(heads, self.engine.fork(seqs[members[0]], len(heads))))
                for i in members:
                    done[i] = end
        for i in range(n):
            if i not in seqs:
                seqs[i] = self.engine.open()
        return done

    def generate(self, prompts: list[list[int]], max_tokens: int = 100, options: SamplingOptions | None = None,
                 stop_ids=None, seed: int = 0, max_batch: int | None = None,
                 on_step: Callable[[int, dict[int, int]], bool | None] | None = None, n: int = 1,
                 share_prefix: bool = False) -> list[GenerationResult]:
        """`n` continuations of every prompt, side by side in the results (request n k + j is continuation j of prompt k, with the
        sampling stream of that number); their prompt goes through the model once. `share_prefix`: so does whatever else the prompts of a
        batch begin with in common."""
        from .step import StepEntry
        if n < 1:
            raise ValueError(f"{n} continuations of a prompt")
        prompts = [p for p in prompts for _ in range(n)]
        options = options or SamplingOptions()
        eng = self.engine
        stop = eng.layout.stop_ids if stop_ids is None else stop_ids
        max_seqs = min(eng.cache.n_slots, max_batch or eng.cache.n_slots)
        batches = plan_batches([len(p) for p in prompts], max_tokens, max_seqs, eng.cache.n_pages, eng.max_positions, n)
        results: list[GenerationResult | None] = [None] * len(prompts)
        # With an engine that keeps per-sequence state records on the device and a sampler that reads
        # them, a step's sampling takes nothing from the host: options and stop set go up once per call,
        # the sequences' seeds once per batch.
        on_device_state = hasattr(self.sampler, "sample_state") and hasattr(getattr(eng, "cache", None), "seq_state")
        if on_device_state:
            self.sampler.begin(options, stop)
        for batch in batches:
            state = BatchState(batch, [prompts[i] for i in batch], max_tokens, stop, eng.max_positions)
            seeds = [seed + r for r in batch]               # one sampling stream per request
            t_ev = [eng.new_event() for _ in range(3)]
            seqs: dict = {}
            try:
                t_ev[0].record()
                live = state.live()
                runs = []
                if n > 1 or share_prefix:
                    runs = shared_runs([s.prompt for s in state.seqs], None if share_prefix else [r // n for r in batch])
                done = self._open(seqs, len(batch), state, runs)
                if on_device_state:
                    eng.cache.seed([seqs[i].slot for i in range(len(batch))], seeds)
                entries = [StepEntry(seqs[i], state.seqs[i].prompt[done[i]:] if done[i] else state.seqs[i].prompt) for i in live]
                if hasattr(eng, "prompt_step"):          # long batches of prompts go through in portions
                    logits, index = eng.prompt_step(entries)
                else:
                    logits = eng.step(entries)
                    index = eng.last_step if on_device_state else None
                fed = [len(state.seqs[i].prompt) for i in live]
                step_no = 0
                # When the engine replays its decode step, the next step is launched with the sampled ids
                # still on the device, before the host reads them: only a stop token can then end a
                # sequence one step "late", and its extra row is dropped.
                pipelined = bool(getattr(eng, "use_graphs", False)) and hasattr(eng, "decode_step_device") \
                    and not options.penalises
                while True:
                    recent = [state.seqs[i].prompt + state.seqs[i].out for i in live] if options.penalises else None
                    if on_device_state:
                        toks_dev = self.sampler.sample_state(logits, eng.cache, index, options, recent)
                    else:
                        toks_dev = self.sampler.sample(logits, options, [seeds[i] for i in live],
                                                       [len(state.seqs[i].out) for i in live], recent)
                    if step_no == 0:
                        t_ev[1].record()
                    ahead = None
                    # the ids start their way to the host before the next step is put on the stream
                    read = self.sampler.begin_read(toks_dev) if pipelined and hasattr(self.sampler, "begin_read") else toks_dev.tolist
                    if pipelined:
                        cont = [j for j, i in enumerate(live) if not state.ends_by_count(i, fed[j])]
                        if cont:
                            rows = toks_dev if len(cont) == len(live) else toks_dev[torch.as_tensor(cont, device=toks_dev.device)]
                            ahead = ([live[j] for j in cont], eng.decode_step_device([seqs[live[j]] for j in cont], rows),
                                     eng.last_step if on_device_state else None)
                    toks = read()
                    for i in state.accept(live, fed, toks):
                        seqs.pop(i).close()
                    if on_step is not None and on_step(step_no, {batch[i]: t for i, t in zip(live, toks)}):
                        for i in state.cancel():
                            seqs.pop(i).close()
                    live = state.live()
                    if not live:
                        break
                    if ahead is not None:
                        keep = [j for j, i in enumerate(ahead[0]) if state.seqs[i].reason is None]
                        if len(keep) == len(ahead[0]):
                            logits, index = ahead[1], ahead[2]
                        else:
                            rows = torch.as_tensor(keep, device=ahead[1].device)
                            logits, index = ahead[1][rows], (ahead[2].rows(rows) if on_device_state else None)
                    else:
                        logits = eng.step([StepEntry(seqs[i], [state.seqs[i].out[-1]]) for i in live])
                        index = eng.last_step if on_device_state else None
                    fed = [1] * len(live)
                    step_no += 1
                t_ev[2].record()
                t_ev[2].synchronize()
                if hasattr(eng, "check_errors"):
                    eng.check_errors()
                pre_ms, dec_ms = t_ev[0].elapsed_time(t_ev[1]), t_ev[1].elapsed_time(t_ev[2])
            finally:
                for s in seqs.values():
                    s.close()
            for s in state.seqs:
                results[s.request] = GenerationResult(s.out, len(s.prompt), s.reason or "cancelled", pre_ms, dec_ms)
        return results
