"""Generation with drafted trees (speculative decoding).

A request's next tokens are guessed from its own tokens: where its last few tokens occurred before, what followed them is a
draft (``lookup_tree``).  Several drafts share their beginnings, so they form a tree, which the model scores in one step
(``ModelRunner.tree_step``).  The accepted tokens are those that the model itself generates, greedily or by sampling with the
uniform numbers that an ordinary step would use, so the drafts change how many steps it takes and not what comes out (but for
the last bits of logits, which another batch gives).

Several samples of one prompt share its pages: the prompt runs once and the request forks (``CacheManager.fork``).  The reference
generates one token a step (demo/llama_infer.cpp:160-200).
"""
from __future__ import annotations

import dataclasses
from typing import Callable, List, Optional, Sequence, Tuple

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

    def generate(self, prompts: Sequence[Sequence[int]], max_new_tokens: int = 16, temperature: float = 0.0, seed: int = 0,
                 ignore_eos: bool = False, samples: int = 1) -> List[List[int]]:
        """``samples`` answers to each prompt, one behind the other.  Answer ``i`` of all is sampled as request ``i`` of an engine is."""
        vocab = self.runner.model.spec.vocab_size
        for p in prompts:
            if not p or any(not 0 <= int(t) < vocab for t in p):
                raise PhotonError(ErrorCode.INVALID_INDEX, f"a prompt needs tokens of the vocabulary of {vocab}")
            if len(p) >= self.runner.max_model_len:
                raise PhotonError(ErrorCode.INVALID_ARGUMENT, f"a prompt of {len(p)} tokens leaves no room in {self.runner.max_model_len}")
        if max_new_tokens < 1 or samples < 1:
            raise PhotonError(ErrorCode.INVALID_ARGUMENT, "at least one new token and one sample are wanted")
        out: List[List[int]] = []
        room = max(1, min(self.options.max_batch_size, self.options.max_sequences) // samples)
        for first in range(0, len(prompts), room):
            group = [[_Sample((first + i) * samples + j, seed, [int(t) for t in p]) for j in range(samples)]
                     for i, p in enumerate(prompts[first:first + room])]
            try:
                self._prefill(group)
                self._decode([s for g in group for s in g], max_new_tokens, temperature, ignore_eos)
            finally:
                for s in (s for g in group for s in g):
                    if self.runner.cache.has_request(s.rid):
                        self.runner.cache.free_request(s.rid)
            out.extend(s.generated for g in group for s in g)
        return out

    def _prefill(self, group: List[List[_Sample]]) -> None:
        """Every prompt but its last token, once, in portions; then the prompt's samples fork from the first."""
        cache, budget = self.runner.cache, self.options.max_num_batched_tokens
        waiting = [(g[0], 0) for g in group]
        for s, _ in waiting:
            cache.add_request(s.rid)
        while waiting:
            entries, left, rest = [], budget, []
            for s, done in waiting:
                n = min(len(s.prompt) - 1 - done, self.options.chunk_size, left)
                if n > 0:
                    entries.append(StepEntry(s.rid, s.prompt[done:done + n]))
                left -= n
                if done + n < len(s.prompt) - 1:
                    rest.append((s, done + n))
            if entries:
                self.runner.step(entries)
            waiting = rest
        for g in group:
            if len(g) > 1:
                cache.fork(g[0].rid, [s.rid for s in g[1:]])

    def _fits(self, sizes: List[Tuple[int, int]]) -> bool:
        """Whether trees of (request, nodes) find their pages."""
        cache = self.runner.cache
        need = [sum(n) for n in zip(*(cache.pages_needed(rid, n) for rid, n in sizes))]
        return all(n <= free for n, free in zip(need, cache.free_pages()))

    def _decode(self, live: List[_Sample], max_new_tokens: int, temperature: float, ignore_eos: bool) -> None:
        eos = self.runner.model.spec.eos_token_ids
        while live:
            # one node each whatever the budget, drafts as far as it goes
            spare = max(0, self.options.max_num_batched_tokens - len(live)) // len(live)
            entries, temps, us = [], [], []
            for s in live:
                tokens = s.prompt + s.generated
                room = min(max_new_tokens - len(s.generated), self.runner.max_model_len - len(tokens) + 1)
                nodes = max(1, min(self.max_nodes, 1 + spare, self.runner.max_model_len - len(tokens) + 1))
                drafted, parents = self.drafter(tokens, nodes, min(self.max_depth, max(0, room - 1)))
                others = [(e.request_id, len(e.tokens)) for e in entries] + [(o.rid, 1) for o in live[len(entries) + 1:]]
                while len(drafted) > 1 and not self._fits(others + [(s.rid, len(drafted))]):
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
                    self.runner.cache.free_request(s.rid)
            live = [s for s in live if s.finish_reason is None]


def generate_drafted(model: str, prompts: Sequence[Sequence[int]], max_new_tokens: int = 16, temperature: float = 0.0, seed: int = 0,
                     options: Optional[EngineOptions] = None, ignore_eos: bool = False, samples: int = 1, max_nodes: int = 16,
                     max_depth: int = 6, drafter: Drafter = lookup_tree) -> List[List[int]]:
    """One call from prompts (token ids) to generated token ids, with drafted trees: ``samples`` answers to each prompt, in order."""
    options = options or EngineOptions()
    generator = DraftingGenerator(build_runner(model, options), options, max_nodes, max_depth, drafter)
    return generator.generate(prompts, max_new_tokens, temperature, seed, ignore_eos, samples)
