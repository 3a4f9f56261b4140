"""Trees of drafted tokens through whole models: logits of every node against the plain implementation of its path, accepted tokens, the cache
behind them, generation with drafts and with several samples."""
import subprocess
import sys
import os

import pytest
import torch

from helpers import ROOT, TINY, TOL, make_finelix_folder, make_model_folder, plain_logits, random_ids, rel_err

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    return {name: make_model_folder(str(tmp_path_factory.mktemp(name)), name) for name in TINY}


def _options(name, dtype, **kw):
    from photon_infer_b200 import EngineOptions
    args = dict(dtype=dtype, block_size=TINY[name]["block_size"], max_cache_tokens=4096, max_sequences=8, chunk_size=24, max_num_batched_tokens=128)
    args.update(kw)
    return EngineOptions(**args)


def _runner(folders, name, dtype, **kw):
    from photon_infer_b200.engine.loading import build_runner
    return build_runner(folders[name], _options(name, dtype, **kw))


def _tree(n, vocab, seed, first):
    import random
    rng = random.Random(seed)
    parents = [-1] + [rng.randint(max(0, i - 6), i - 1) for i in range(1, n)]
    return [first] + [rng.randrange(vocab) for _ in range(n - 1)], parents


def _path(tokens, parents, i):
    out = []
    while i >= 0:
        out.append(tokens[i])
        i = parents[i]
    return out[::-1]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", list(TINY))
def test_every_nodes_logits_are_its_paths(folders, name, dtype):
    """Two requests, one of them without cached tokens, trees of one node to more than a mask word has bits; then a step of ordinary tokens behind the
    accepted nodes sees the cache as if they had been decoded one by one."""
    from photon_infer_b200.engine.runner import StepEntry, TreeEntry
    runner = _runner(folders, name, dtype)
    vocab = TINY[name]["config"]["vocab_size"]
    prompts = {"a": random_ids(53, vocab, 1), "b": random_ids(1, vocab, 2), "c": random_ids(90, vocab, 3)}
    cached = {}
    for rid, p in prompts.items():
        runner.cache.add_request(rid)
        if len(p) > 1:
            runner.step([StepEntry(rid, p[:-1])])
        cached[rid] = p[:-1]
    for round_, sizes in enumerate(((37, 5, 1), (3, 9, 12))):
        trees = {rid: _tree(n, vocab, 10 * round_ + i, prompts[rid][-1]) for i, (rid, n) in enumerate(zip(prompts, sizes))}
        # one of the nodes carries what the model would generate, so that some paths are longer than the first node
        for rid, (tokens, parents) in trees.items():
            if len(tokens) > 2:
                best = int(plain_logits(folders[name], cached[rid] + [tokens[0]])[-1].argmax())
                tokens[[i for i, p in enumerate(parents) if p == 0][-1]] = best
        result = runner.tree_step([TreeEntry(rid, *trees[rid]) for rid in prompts])
        at = 0
        for s, rid in enumerate(prompts):
            tokens, parents = trees[rid]
            for i in range(len(tokens)):
                want = plain_logits(folders[name], cached[rid] + _path(tokens, parents, i))[-1:]
                assert rel_err(result.logits[at + i:at + i + 1].cpu(), want) <= TOL[dtype], (rid, i)
            path, given = result.paths[s], result.tokens[s]
            assert path[0] == 0 and len(given) == len(path)
            for j, node in enumerate(path):
                assert given[j] == int(result.logits[at + node].argmax())
                if j + 1 < len(path):
                    assert parents[path[j + 1]] == node and tokens[path[j + 1]] == given[j]
            assert not any(p == path[-1] and t == given[-1] for t, p in zip(tokens, parents))
            cached[rid] = cached[rid] + [tokens[i] for i in path]
            prompts[rid] = cached[rid] + [given[-1]]
            assert runner.cache.length(rid) == len(cached[rid])
            at += len(tokens)
        runner.cache.check_consistency()
    assert any(len(p) > 1 for p in result.paths)
    more = {rid: random_ids(4, vocab, 30) for rid in prompts}
    got = runner.step([StepEntry(rid, more[rid], [0, 3]) for rid in prompts]).logits.cpu()
    want = torch.cat([plain_logits(folders[name], cached[rid] + more[rid])[[-4, -1]] for rid in prompts])
    assert rel_err(got, want) <= TOL[dtype]


def _attention(kind, heads, kv_heads, dim, size=None, **more):
    mixer = dict(heads=heads, kv_heads=kv_heads, dim=dim, vdim=dim, scale=0.2, **more)
    if size:
        mixer["mask"] = dict(size=size)
    return dict(type=kind, mixer=mixer, mlp=None)


# sinks, softcaps, gates, windows and a looped block; heads of 64 and 128 and others; pages of 16 and 8
_FEKOPEL = {
    "wide": dict(width=64, page=16, loop=dict(start=0, stop=2, times=2), layers=[
        _attention("attention_2", 2, 1, 64, 40, rot=dict(base=5000.0, dims=16), softcap=6.0), _attention("attention", 4, 2, 64, 24),
        _attention("attention", 2, 1, 128), _attention("attention_2", 3, 3, 128, softcap=15.0)]),
    "odd": dict(width=50, page=8, loop=None, layers=[
        _attention("attention_2", 3, 1, 10, 3, rot=dict(base=777.0, dims=6), softcap=9.0), _attention("attention", 5, 5, 6, 37),
        _attention("attention_2", 2, 2, 18)]),
}


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", list(_FEKOPEL))
def test_sinks_softcaps_and_gates(tmp_path, name, dtype):
    from helpers import fekopel_plain_logits
    from photon_infer_b200 import EngineOptions
    from photon_infer_b200.engine.loading import build_runner
    from photon_infer_b200.engine.runner import StepEntry, TreeEntry
    from photon_infer_b200.weights import write_random_model
    t = _FEKOPEL[name]
    folder = str(tmp_path / name)
    write_random_model(folder, dict(architecture="Fekopel", vocab=150, width=t["width"], norm=dict(eps=1e-5), layers=t["layers"],
                                    loop=t["loop"]), seed=31, init_std=0.1, norm_std=0.1, dtype="bfloat16")
    runner = build_runner(folder, EngineOptions(dtype=dtype, block_size=t["page"], max_cache_tokens=1024, max_sequences=4))
    cached = {"a": random_ids(61, 150, 1), "b": random_ids(6, 150, 2)}
    for rid, p in cached.items():
        runner.cache.add_request(rid)
        runner.step([StepEntry(rid, p)])
    for sizes in ((35, 4), (2, 40)):
        trees = [_tree(n, 150, n, 7) for n in sizes]
        result = runner.tree_step([TreeEntry(rid, *tree) for rid, tree in zip(cached, trees)])
        at = 0
        for s, ((rid, ids), (tokens, parents)) in enumerate(zip(list(cached.items()), trees)):
            for i in range(len(tokens)):
                want = fekopel_plain_logits(folder, ids + _path(tokens, parents, i))[-1:]
                assert rel_err(result.logits[at + i:at + i + 1].cpu(), want) <= TOL[dtype], (rid, i)
            cached[rid] = ids + [tokens[i] for i in result.paths[s]]
            at += len(tokens)


def _oracle(folder, wrong):
    """A drafter that knows the greedy continuation, hides it between wrong siblings and is mistaken at every ``wrong``-th place."""
    from plain.llama_plain import PlainLlama
    model = PlainLlama.from_folder(folder)

    def draft(tokens, max_nodes, max_depth):
        tree, parents, node, ids = [tokens[-1]], [-1], 0, list(tokens)
        for _ in range(max_depth):
            best = int(torch.argmax(model.logits(ids)[-1]))
            for t in (best ^ 1, best ^ 2, best):
                if len(tree) < max_nodes and t < model.logits(ids).shape[1]:
                    tree.append(t)
                    parents.append(node)
            if tree[-1] != best or len(ids) % wrong == 0:
                break
            node = len(tree) - 1
            ids.append(best)
        return tree, parents
    return draft


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["tiny_a", "tiny_d"])
def test_drafts_change_the_steps_and_not_the_tokens(folders, name, dtype):
    from photon_infer_b200 import DraftingGenerator
    from test_gpu_engine import _plain_greedy_checked
    vocab = TINY[name]["config"]["vocab_size"]
    prompts = [random_ids(n, vocab, seed=n) for n in (1, 9, 33)]
    options = _options(name, dtype)
    runner = _runner(folders, name, dtype)
    generator = DraftingGenerator(runner, options, max_nodes=12, max_depth=4, drafter=_oracle(folders[name], 5))
    out = generator.generate(prompts, 14, ignore_eos=True)
    for p, got in zip(prompts, out):
        assert len(got) == 14
        _plain_greedy_checked(folders[name], p, got, dtype)
    assert generator.stats.generated == 42 and generator.stats.steps <= 10          # 14 steps without drafts
    assert runner.cache.live_requests() == [] and runner.cache.free_pages() == [g.num_pages for g in runner.cache.groups]
    if dtype == "float32":
        from plain.llama_plain import PlainLlama
        assert out[1] == PlainLlama.from_folder(folders[name]).greedy(prompts[1], 14)


def test_sampling_is_the_engines(folders):
    """With a temperature the tokens are those of ordinary steps with the same numbers (32 bits), drafts accepted or not; samples of a prompt, which
    fork from one another, are the engine's requests of the same ids."""
    from photon_infer_b200 import ContinuousBatchEngine, DraftingGenerator
    name = "tiny_b"
    vocab = TINY[name]["config"]["vocab_size"]
    prompts = [random_ids(n, vocab, seed=n) for n in (21, 13)]
    engine = ContinuousBatchEngine(folders[name], _options(name, "float32"))
    ids = [engine.add_request(p, 12, temperature=0.9, seed=4, ignore_eos=True) for p in prompts for _ in range(3)]
    want = engine.run_until_complete()
    known = {tuple(p): [want[i] for i in ids[3 * k:3 * k + 3]] for k, p in enumerate(prompts)}

    def draft(tokens, max_nodes, max_depth):
        tree, parents = [tokens[-1]], [-1]
        for p, answers in known.items():
            for a in answers:
                full = list(p) + a
                if full[:len(tokens)] == list(tokens):
                    node = 0
                    for t in full[len(tokens):len(tokens) + max_depth]:
                        if len(tree) == max_nodes:
                            break
                        tree.append(t)
                        parents.append(node)
                        node = len(tree) - 1
        return tree, parents
    options = _options(name, "float32")
    generator = DraftingGenerator(_runner(folders, name, "float32"), options, 10, 3, draft)
    got = generator.generate(prompts, 12, temperature=0.9, seed=4, ignore_eos=True, samples=3)
    assert got == [want[i] for i in ids]
    assert generator.stats.steps < 10


def test_few_pages(folders):
    """Drafts shrink where pages run out; what is generated does not change."""
    from photon_infer_b200 import DraftingGenerator
    name, prompt = "tiny_a", [3, 4, 5, 6] * 6
    ample, tight = (_options(name, "float32", max_cache_tokens=n) for n in (4096, 80))
    want, got = (DraftingGenerator(_runner(folders, name, "float32", max_cache_tokens=o.max_cache_tokens), o, 40, 6,
                                   lambda tokens, n, d: ([tokens[-1]] + [1] * (n - 1), [-1] + [0] * (n - 1))).generate([prompt, prompt[:9]], 10, ignore_eos=True)
                 for o in (ample, tight))
    assert got == want


def test_end_of_sequence_and_length(folders):
    from photon_infer_b200 import ContinuousBatchEngine, generate_drafted
    name = "tiny_c"
    vocab = TINY[name]["config"]["vocab_size"]
    prompt = random_ids(1010, vocab, 5)                     # the model ends at 1,024 tokens
    got = generate_drafted(folders[name], [prompt], 40, options=_options(name, "float32"), ignore_eos=True)
    assert len(got[0]) == 14
    engine = ContinuousBatchEngine(folders[name], _options(name, "float32"))
    rid = engine.add_request(prompt, 40, ignore_eos=True)
    assert engine.run_until_complete()[rid] == got[0]


def test_command_line(folders):
    cmd = [sys.executable, os.path.join(ROOT, "bin", "llama_infer"), folders["tiny_a"], "cuda", "--prompt-ids", "5,6,7,5,6", "--max-new-tokens", "9",
           "--temperature", "0", "--ignore-eos", "--dtype", "float32", "--num-blocks", "32"]
    plain = subprocess.run(cmd, capture_output=True, text=True)
    drafted = subprocess.run(cmd + ["--draft-nodes", "8", "--samples", "2"], capture_output=True, text=True)
    assert plain.returncode == 0 and drafted.returncode == 0, plain.stderr + drafted.stderr
    tokens = plain.stdout.split(":")[1].split()
    lines = drafted.stdout.strip().splitlines()
    assert len(lines) == 2 and all(line.split(":")[1].split() == tokens for line in lines)
    refused = subprocess.run(cmd + ["--samples", "2"], capture_output=True, text=True)
    assert refused.returncode == 1 and "--draft-nodes" in refused.stderr


def test_refusals(folders, tmp_path):
    from photon_infer_b200 import EngineOptions
    from photon_infer_b200.engine.loading import build_runner
    from photon_infer_b200.engine.runner import TreeEntry
    from photon_infer_b200.errors import ErrorCode, PhotonError
    runner = _runner(folders, "tiny_a", "float32", max_cache_tokens=64, max_model_len=40)
    runner.cache.add_request("a")

    def refused(code, entries, **kw):
        with pytest.raises(PhotonError) as e:
            runner.tree_step(entries, **kw)
        assert e.value.code == code
        assert runner.cache.length("a") == 0 and runner.cache.free_pages() == [4]
    assert runner.tree_step([]).tokens == []
    refused(ErrorCode.INVALID_STATE, [TreeEntry("x", [1], [-1])])
    refused(ErrorCode.INVALID_ARGUMENT, [TreeEntry("a", [1], [-1])] * 2)
    refused(ErrorCode.INVALID_ARGUMENT, [TreeEntry("a", [1, 2], [-1])])
    refused(ErrorCode.INVALID_ARGUMENT, [TreeEntry("a", [1, 2], [-1, 1])])
    refused(ErrorCode.INVALID_ARGUMENT, [TreeEntry("a", [], [])])
    refused(ErrorCode.INVALID_ARGUMENT, [TreeEntry("a", [1] * 41, [-1] + [0] * 40)])
    refused(ErrorCode.INVALID_ARGUMENT, [TreeEntry("a", [1], [-1])], sampling=([1.0], []))
    runner.cache.add_request("b")
    runner.cache.extend("b", 40)
    with pytest.raises(PhotonError) as e:
        runner.tree_step([TreeEntry("a", [1] * 20, [-1] + [0] * 19)])
    assert e.value.code == ErrorCode.OUT_OF_MEMORY and runner.cache.free_pages() == [1]
    folder = make_finelix_folder(str(tmp_path / "fx"), "fx_a")
    other = build_runner(folder, EngineOptions(dtype="float32", block_size=16, max_cache_tokens=64))
    other.cache.add_request("a")
    with pytest.raises(PhotonError) as e:
        other.tree_step([TreeEntry("a", [1], [-1])])
    assert e.value.code == ErrorCode.UNSUPPORTED_MODEL
