"""Generation with drafted trees where the cache is smaller than the requests together, on the host: a model that is a function of a request's text stands in for
the kernels, so that the answers are known whatever waits for what."""
import types

import pytest
import torch

from photon_infer_b200 import EngineOptions
from photon_infer_b200.cache import CacheManager
from photon_infer_b200.engine.drafting import DraftingGenerator
from photon_infer_b200.engine.runner import TreeStepResult
from photon_infer_b200.errors import ErrorCode, PhotonError
from photon_infer_b200.parts.base import PagedCacheSpec
from photon_infer_b200.sampling.sampler import uniform

VOCAB, EOS = 97, 3
FULL, WINDOW = PagedCacheSpec(1, 8, None), PagedCacheSpec(1, 8, 9)


def _next(text, u=0.0):
    x = 17
    for t in text:
        x = (x * 31 + t + 7) % 1000003
    return int(x + 1000 * u) % VOCAB


class _Cache(CacheManager):
    """Keeps each request's cached text beside its pages."""

    def __init__(self, *a):
        super().__init__(*a)
        self.text = {}

    def add_request(self, rid):
        self.text[rid] = []
        return super().add_request(rid)

    def fork(self, rid, new_rids):
        super().fork(rid, new_rids)
        for new in new_rids:
            self.text[new] = list(self.text[rid])

    def free_request(self, rid):
        super().free_request(rid)
        del self.text[rid]


class _Runner:
    def __init__(self, pages, page_size=4, max_sequences=16, specs=(FULL,), max_model_len=200):
        self.cache = _Cache([(s, None) for s in specs], [None] * len(specs), page_size, pages, max_sequences, torch.float32, None)
        self.model = types.SimpleNamespace(spec=types.SimpleNamespace(vocab_size=VOCAB, eos_token_ids=(EOS,)))
        self.max_model_len = max_model_len
        self.most = 0

    def _take(self, sizes):
        need = [sum(n) for n in zip(*(self.cache.pages_needed(rid, n) for rid, n in sizes))]
        if any(n > f for n, f in zip(need, self.cache.free_pages())):
            raise PhotonError(ErrorCode.OUT_OF_MEMORY, "no pages")
        for rid, n in sizes:
            self.cache.extend(rid, n)
        self.most = max(self.most, len(sizes))

    def step(self, entries):
        self._take([(e.request_id, len(e.tokens)) for e in entries])
        for e in entries:
            self.cache.text[e.request_id] += e.tokens
            self.cache.commit(e.request_id, len(e.tokens))

    def tree_step(self, entries, sampling=None):
        self._take([(e.request_id, len(e.tokens)) for e in entries])
        result, at = TreeStepResult([], [], None), 0
        for e in entries:
            text = self.cache.text[e.request_id]
            assert len(text) == self.cache.length(e.request_id)
            node, path, given = 0, [], []
            while node is not None:
                text.append(e.tokens[node])
                path.append(node)
                given.append(_next(text, sampling[1][at + node] if sampling else 0.0))
                node = next((i for i in range(node + 1, len(e.tokens)) if e.parents[i] == node and e.tokens[i] == given[-1]), None)
            result.paths.append(path)
            result.tokens.append(given)
            self.cache.commit_kept(e.request_id, len(path))
            at += len(e.tokens)
        return result


def _want(prompt, n, rid, temperature, seed, ignore_eos):
    text = list(prompt)
    while len(text) - len(prompt) < n:
        text.append(_next(text, uniform(seed, rid, len(text) - len(prompt)) if temperature > 0 else 0.0))
        if text[-1] == EOS and not ignore_eos:
            break
    return text[len(prompt):]


def _knowing(tokens, max_nodes, max_depth):
    """A drafter that knows the greedy continuation and puts wrong tokens beside it."""
    tree, parents, node, text = [tokens[-1]], [-1], 0, list(tokens)
    for _ in range(max_depth):
        text.append(_next(text))
        for t in (text[-1] ^ 1, text[-1]):
            if len(tree) < max_nodes:
                tree.append(t)
                parents.append(node)
        if tree[-1] != text[-1]:
            break
        node = len(tree) - 1
    return tree, parents


def _prompts(lengths):
    return [[(5 * i + 3 * j + 1) % VOCAB for j in range(n)] for i, n in enumerate(lengths)]


@pytest.mark.parametrize("specs", [(FULL,), (WINDOW,), (FULL, WINDOW)])
@pytest.mark.parametrize("samples", [1, 3])
@pytest.mark.parametrize("pages", [11, 14, 20, 33, 400])
@pytest.mark.parametrize("temperature", [0.0, 0.8])
@pytest.mark.parametrize("chunk,budget", [(256, 2048), (7, 16)])
def test_requests_that_do_not_fit_together(specs, samples, pages, temperature, chunk, budget):
    """Prompts of which the largest alone fits, up to all of them: the same answers, every page given back."""
    lengths = [1, 23, 8, 30, 2, 17, 12]                     # 30 + 12 tokens and a draft: 11 pages of 4
    runner = _Runner(pages, specs=specs)
    options = EngineOptions(max_batch_size=9, max_sequences=16, chunk_size=chunk, max_num_batched_tokens=budget)
    generator = DraftingGenerator(runner, options, 6, 3, _knowing)
    prompts = _prompts(lengths)
    got = generator.generate(prompts, 12, temperature, seed=5, ignore_eos=True, samples=samples)
    assert got == [_want(p, 12, i * samples + j, temperature, 5, True) for i, p in enumerate(prompts) for j in range(samples)]
    assert generator.finish_reasons == ["length"] * len(got) and runner.most <= 9
    assert runner.cache.live_requests() == [] and runner.cache.free_pages() == [pages] * len(specs)
    runner.cache.check_consistency()


def test_one_that_does_not_fit_alone():
    """It ends with what it has, or with nothing where its prompt does not fit; the others' answers are whole, and they may end at a token of their own."""
    prompts = _prompts([9, 60, 26, 5])
    generator = DraftingGenerator(_Runner(8), EngineOptions(max_batch_size=4, max_sequences=4), 6, 3, _knowing)
    got = generator.generate(prompts, 15, ignore_eos=True)
    whole = [_want(p, 15, i, 0.0, 0, True) for i, p in enumerate(prompts)]
    assert got[0] == whole[0] and got[3] == whole[3] and got[1] == []
    assert 0 < len(got[2]) < 15 and got[2] == whole[2][:len(got[2])]
    assert generator.finish_reasons == ["length", "out_of_memory", "out_of_memory", "length"]
    assert generator.runner.cache.free_pages() == [8]
    want = [_want(p, 150, i, 0.0, 0, False) for i, p in enumerate(_prompts([4, 6]))]
    generator = DraftingGenerator(_Runner(100), EngineOptions(), 6, 3, _knowing)
    assert generator.generate(_prompts([4, 6]), 150) == want
    assert generator.finish_reasons == ["eos" if w[-1] == EOS else "length" for w in want]


def test_more_samples_than_slots():
    """Samples run as many at a time as the engine's bounds allow."""
    runner = _Runner(60, max_sequences=4)
    generator = DraftingGenerator(runner, EngineOptions(max_batch_size=3, max_sequences=4), 6, 3, _knowing)
    got = generator.generate(_prompts([9, 6]), 7, 0.9, seed=2, ignore_eos=True, samples=10)
    assert got == [_want(p, 7, 10 * i + j, 0.9, 2, True) for i, p in enumerate(_prompts([9, 6])) for j in range(10)] and runner.most <= 3


@pytest.mark.parametrize("drafted", [([], []), ([8], [-1]), ([8, 9], [-1, 0])])
def test_drafts_that_do_not_begin_with_the_last_token(drafted):
    """A tree that would put another token, or none, in the place of the request's last one is refused; nothing stays taken."""
    runner = _Runner(20)
    generator = DraftingGenerator(runner, EngineOptions(), 6, 3, lambda text, n, d: drafted)
    with pytest.raises(PhotonError) as e:
        generator.generate([[1, 2, 7]], 4, ignore_eos=True)
    assert e.value.code == ErrorCode.INVALID_ARGUMENT and runner.cache.live_requests() == [] and runner.cache.free_pages() == [20]
