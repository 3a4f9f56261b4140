"""Generation with drafted trees (speculative decoding).

A request's next tokens are guessed from its own tokens: where its last few tokens occurred before, what followed them is a
draft (``lookup_tree``).  Several drafts share their beginnings, so they form a tree, which the model scores in one step
(``ModelRunner.tree_step``).  The accepted tokens are those that the model itself generates, greedily or by sampling with the
uniform numbers that an ordinary step would use, so the drafts change how many steps it takes and not what comes out (but for
the last bits of logits, which another batch gives).

Several samples of one prompt share its pages: the prompt runs once and the request forks (``CacheManager.fork``).  Where pages run out the
request that came last waits, as in the scheduler: its pages are freed and its tokens are computed again later.  The reference
generates one token a step (demo/llama_infer.cpp:160-200).
"""
from __future__ import annotations

import collections
import dataclasses
from typing import Callable, Deque, List, Optional, Sequence, Tuple

from ..config.engine_options import EngineOptions
from ..errors import ErrorCode, PhotonError
from ..sampling.sampler import uniform
from .loading import build_runner
from .runner import ModelRunner, StepEntry, TreeEntry

#: A drafter: (a request's tokens, most nodes, most levels below the first node) -> (tokens, parents) of a tree whose first
#: node is the request's last token.
Drafter = Callable[[Sequence[int], int, int], Tuple[List[int], List[int]]]


def lookup_tree(tokens: Sequence[int], max_nodes: int, max_depth: int, ngram: int = 3) -> Tuple[List[int], List[int]]:
    """A tree of what followed earlier occurrences of the last ``ngram`` tokens (then of fewer), the latest occurrence first."""
    tree, parents = [tokens[-1]], [-1]
    children = {}
    for n in range(min(ngram, len(tokens) - 1), 0, -1):
        last = list(tokens[-n:])
        for at in range(len(tokens) - n - 1, -1, -1):
            if tokens[at + n - 1] != last[-1] or list(tokens[at:at + n]) != last:
                continue
            node = 0
            for t in tokens[at + n: at + n + max_depth]:
                if (node, t) not in children:
                    if len(tree) >= max_nodes:
                        return tree, parents
                    children[node, t] = len(tree)
                    tree.append(t)
                    parents.append(node)
                node = children[node, t]
    return tree, parents


@dataclasses.dataclass
class _Sample:
    rid: int
    seed: int
    prompt: List[int]
    generated: List[int] = dataclasses.field(default_factory=list)
    finish_reason: Optional[str] = None

    def tokens(self) -> List[int]:
        return self.prompt + self.generated


#: Samples of one prompt that run it once and fork; one that had to wait is a group of its own.
_Group = List[_Sample]


@dataclasses.dataclass
class DraftStats:
    steps: int = 0                      # steps of trees
    nodes: int = 0                      # tokens they ran
    generated: int = 0                  # tokens they gave


class DraftingGenerator:
    """Runs prompts to generated tokens with drafted trees of up to ``max_nodes`` nodes, the request's last token among them."""

    def __init__(self, runner: ModelRunner, options: EngineOptions, max_nodes: int = 16, max_depth: int = 6,
                 drafter: Drafter = lookup_tree):
        if max_nodes < 1 or max_depth < 0:
            raise PhotonError(ErrorCode.INVALID_ARGUMENT, "a tree needs at least one node and no fewer than 0 levels below it")
        self.runner, self.options, self.drafter = runner, options, drafter
        self.max_nodes, self.max_depth = max_nodes, max_depth
        self.stats = DraftStats()
        self.finish_reasons: List[str] = []     # of the last call's answers: "eos", "length", "model_len" or "out_of_memory"

    def generate(self, prompts: Sequence[Sequence[int]], max_new_tokens: int = 16, temperature: float = 0.0, seed: int = 0,
                 ignore_eos: bool = False, samples: int = 1) -> List[List[int]]:
        """``samples`` answers to each prompt, one behind the other.  Answer ``i`` of all is sampled as request ``i`` of an engine is.  An answer that
        does not fit the cache although nothing else runs ends there, as in an engine (``finish_reasons``)."""
        vocab = self.runner.model.spec.vocab_size
        for p in prompts:
            if not p or any(not 0 <= int(t) < vocab for t in p):
                raise PhotonError(ErrorCode.INVALID_INDEX, f"a prompt needs tokens of the vocabulary of {vocab}")
            if len(p) >= self.runner.max_model_len:
                raise PhotonError(ErrorCode.INVALID_ARGUMENT, f"a prompt of {len(p)} tokens leaves no room in {self.runner.max_model_len}")
        if max_new_tokens < 1 or samples < 1:
            raise PhotonError(ErrorCode.INVALID_ARGUMENT, "at least one new token and one sample are wanted")
        groups: List[_Group] = [[_Sample(i * samples + j, seed, [int(t) for t in p]) for j in range(samples)] for i, p in enumerate(prompts)]
        answers = [s for g in groups for s in g]
        waiting: Deque[_Group] = collections.deque(groups)
        try:
            while waiting:
                self._decode(self._prefill(waiting), waiting, max_new_tokens, temperature, ignore_eos)
        finally:
            for s in answers:
                if self.runner.cache.has_request(s.rid):
                    self.runner.cache.free_request(s.rid)
        self.finish_reasons = [s.finish_reason for s in answers]
        return [s.generated for s in answers]

    def _prefill(self, waiting: Deque[_Group]) -> List[_Sample]:
        """As many groups as may run together: every group's tokens but the last, once, in portions; then its samples fork from the first.  Returns
        those that run.  What finds no pages goes back to ``waiting``, the last group first."""
        cache, limit = self.runner.cache, min(self.options.max_batch_size, self.options.max_sequences)
        batch: List[_Group] = []
        while waiting and (not batch or sum(len(g) for g in batch) + len(waiting[0]) <= limit):
            batch.append(waiting.popleft())
            cache.add_request(batch[-1][0].rid)

        def last_waits() -> None:
            g = batch.pop()
            cache.free_request(g[0].rid)
            waiting.appendleft(g)

        todo = [(g, 0) for g in batch]
        while todo:
            entries, left, rest = [], self.options.max_num_batched_tokens, []
            taken = [0] * len(cache.groups)         # pages of the step's entries
            for g, done in todo:
                if not any(g is b for b in batch):
                    continue                        # it waits
                s, tokens = g[0], g[0].tokens()[:-1]
                n = min(len(tokens) - done, self.options.chunk_size, left)
                if n > 0:
                    need = [a + b for a, b in zip(taken, cache.pages_needed(s.rid, n))]
                    while not self._free(need) and batch[-1] is not g:
                        last_waits()
                    if not self._free(need):
                        last_waits()
                        if not batch:               # alone and still too large for the pool
                            for s in waiting.popleft():
                                s.finish_reason = "out_of_memory"
                        continue
                    entries.append(StepEntry(s.rid, tokens[done:done + n]))
                    taken = need
                left -= n
                if done + n < len(tokens):
                    rest.append((g, done + n))
            if entries:
                self.runner.step(entries)
            todo = rest
        live: List[_Sample] = []
        at = 0
        while at < len(batch):
            g = batch[at]
            at += 1
            while self._forks(g[0].rid, len(g) - 1, limit - len(live) - 1) < len(g) - 1 and at < len(batch):
                last_waits()
            n = self._forks(g[0].rid, len(g) - 1, limit - len(live) - 1)
            if n > 0:
                cache.fork(g[0].rid, [s.rid for s in g[1:n + 1]])
            live += g[:n + 1]
            if n + 1 < len(g):
                waiting.appendleft(g[n + 1:])
        return live

    def _forks(self, rid, wanted: int, room: int) -> int:
        """How many forks of a request find their pages and slots, up to ``wanted`` and ``room``."""
        cache = self.runner.cache
        n = min(wanted, max(0, room), cache.states.num_free)
        for g, free in zip(cache.groups, cache.free_pages()):
            each = g.pages_to_fork(cache.length(rid))
            n = min(n, free // each if each else n)
        return n

    def _free(self, need: List[int]) -> bool:
        """Whether as many pages are free in every cache group."""
        return all(n <= free for n, free in zip(need, self.runner.cache.free_pages()))

    def _decode(self, live: List[_Sample], waiting: Deque[_Group], max_new_tokens: int, temperature: float, ignore_eos: bool) -> None:
        eos, cache = self.runner.model.spec.eos_token_ids, self.runner.cache
        while live:
            ones = [cache.pages_needed(s.rid, 1) for s in live]
            while not self._free([sum(n) for n in zip(*ones)]):
                s = live.pop()
                ones.pop()
                cache.free_request(s.rid)
                if not live:                        # alone and still too large for the pool
                    s.finish_reason = "out_of_memory"
                    return
                waiting.appendleft([s])
            taken = [sum(n) for n in zip(*ones)]    # pages of the step: one node each, and the drafts so far
            # one node each whatever the budget, drafts as far as it goes
            spare = max(0, self.options.max_num_batched_tokens - len(live)) // len(live)
            entries, temps, us = [], [], []
            for s, one in zip(live, ones):
                tokens = s.tokens()
                room = min(max_new_tokens - len(s.generated), self.runner.max_model_len - len(tokens) + 1)
                nodes = max(1, min(self.max_nodes, 1 + spare, self.runner.max_model_len - len(tokens) + 1))
                drafted, parents = self.drafter(tokens, nodes, min(self.max_depth, max(0, room - 1)))
                if not drafted or drafted[0] != tokens[-1]:
                    raise PhotonError(ErrorCode.INVALID_ARGUMENT, f"the drafter's tree for request {s.rid} begins with {list(drafted[:1])}, not with its last token, {tokens[-1]}")
                while len(drafted) > 1:
                    need = [t - a + b for t, a, b in zip(taken, one, cache.pages_needed(s.rid, len(drafted)))]
                    if self._free(need):
                        taken = need
                        break
                    drafted, parents = drafted[:len(drafted) // 2], parents[:len(drafted) // 2]     # few pages are left
                entries.append(TreeEntry(s.rid, drafted, parents))
                depth: List[int] = []
                for p in parents:
                    depth.append(0 if p < 0 else depth[p] + 1)
                temps.append(temperature)
                us.extend(uniform(s.seed, s.rid, len(s.generated) + d) if temperature > 0 else 0.0 for d in depth)
            result = self.runner.tree_step(entries, sampling=(temps, us) if temperature > 0 else None)
            self.stats.steps += 1
            self.stats.nodes += sum(len(e.tokens) for e in entries)
            for s, got in zip(live, result.tokens):
                for t in got:
                    s.generated.append(t)
                    self.stats.generated += 1
                    if not ignore_eos and t in eos:
                        s.finish_reason = "eos"
                    elif len(s.generated) >= max_new_tokens:
                        s.finish_reason = "length"
                    elif len(s.prompt) + len(s.generated) >= self.runner.max_model_len:
                        s.finish_reason = "model_len"
                    if s.finish_reason is not None:
                        break
                if s.finish_reason is not None:
                    cache.free_request(s.rid)
            live = [s for s in live if s.finish_reason is None]


def generate_drafted(model: str, prompts: Sequence[Sequence[int]], max_new_tokens: int = 16, temperature: float = 0.0, seed: int = 0,
                     options: Optional[EngineOptions] = None, ignore_eos: bool = False, samples: int = 1, max_nodes: int = 16,
                     max_depth: int = 6, drafter: Drafter = lookup_tree) -> List[List[int]]:
    """One call from prompts (token ids) to generated token ids, with drafted trees: ``samples`` answers to each prompt, in order."""
    options = options or EngineOptions()
    generator = DraftingGenerator(build_runner(model, options), options, max_nodes, max_depth, drafter)
    return generator.generate(prompts, max_new_tokens, temperature, seed, ignore_eos, samples)
