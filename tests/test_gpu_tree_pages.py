"""Generation with drafted trees through a whole model whose cache holds a part of the requests, beside the engine with ample and with as little cache."""
import pytest

from helpers import TINY, make_model_folder, random_ids
from test_gpu_tree_model import _options

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    return {name: make_model_folder(str(tmp_path_factory.mktemp(name)), name) for name in TINY}


@pytest.mark.parametrize("name", list(TINY))
@pytest.mark.parametrize("temperature", [0.0, 0.9])
def test_prompts_that_do_not_fit_together(folders, name, temperature):
    """32 bits: a request that waited is computed again, to the same tokens."""
    from photon_infer_b200 import ContinuousBatchEngine, DraftingGenerator
    from photon_infer_b200.engine.loading import build_runner
    vocab, page = TINY[name]["config"]["vocab_size"], TINY[name]["block_size"]
    prompts = [random_ids(n, vocab, seed=n) for n in (5, 61, 33, 12, 50)]
    pages = -(-(61 + 14) // page) + 2                       # the largest request, a draft, and little more
    answers = []
    for num_blocks in (None, pages):
        options = _options(name, "float32", num_blocks=num_blocks)
        engine = ContinuousBatchEngine(folders[name], options)
        ids = [engine.add_request(p, 14, temperature=temperature, seed=4, ignore_eos=True) for p in prompts for _ in range(2)]
        out = engine.run_until_complete()
        answers.append([out[i] for i in ids])
        runner = build_runner(folders[name], options)
        generator = DraftingGenerator(runner, options, 8, 3)
        answers.append(generator.generate(prompts, 14, temperature=temperature, seed=4, ignore_eos=True, samples=2))
        assert generator.finish_reasons == ["length"] * 10
        assert runner.cache.live_requests() == [] and runner.cache.free_pages() == [g.num_pages for g in runner.cache.groups]
    assert answers[1] == answers[0] and answers[3] == answers[0]


@pytest.mark.parametrize("depth", [0, -1])
def test_a_depth_below_one_is_refused(folders, depth):
    from photon_infer_b200.engine.loading import build_runner
    from photon_infer_b200.engine.runner import TreeEntry
    from photon_infer_b200.errors import ErrorCode, PhotonError
    runner = build_runner(folders["tiny_a"], _options("tiny_a", "float32"))
    runner.cache.add_request("a")
    free = runner.cache.free_pages()
    with pytest.raises(PhotonError) as e:
        runner.tree_step([TreeEntry("a", [1, 2], [-1, 0])], depth=depth)
    assert e.value.code == ErrorCode.INVALID_ARGUMENT and runner.cache.free_pages() == free
