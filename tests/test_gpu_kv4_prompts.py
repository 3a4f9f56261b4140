"""Prompt portions in bfloat16 both ways: pages laid out for the tcgen05 kernel, and the codes eight rows at a time, whatever the rule says."""
import pytest
import torch

import test_gpu_kv4_attention as few

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[False, True], ids=["laid-out", "codes"])
def way(request, monkeypatch):
    from photon_infer_b200.kernels import ops
    monkeypatch.setattr(ops, "_kv4_few", lambda *sizes: request.param)


@pytest.mark.parametrize("count,held", [([40], [40]), ([17, 1, 33], [200, 90, 33]), ([1, 70, 0, 5], [600, 450, 3, 5]), ([130], [1000])])
@pytest.mark.parametrize("n_q,n_kv,d,page", [(8, 2, 64, 16), (4, 1, 128, 8), (2, 2, 64, 32)])
def test_prompts(way, n_q, n_kv, d, page, count, held):
    few.test_prompts(torch.bfloat16, n_q, n_kv, d, page, count, held)


@pytest.mark.parametrize("more", [dict(window=50), dict(softcap=5.0), dict(sink=True)])
def test_masks(way, more):
    few.test_prompts_with_masks(more)


def test_slices_and_bounds(way, monkeypatch):
    few.test_prompts_in_slices(monkeypatch)
    few.test_fewer_tokens_than_announced()


def test_strides_and_a_missing_page(way):
    few.test_strides_and_rows_behind_the_last(torch.bfloat16, 40)
    few.test_a_missing_page(torch.bfloat16, 40)


@pytest.mark.parametrize("n_q,n_kv,d,page", [(8, 2, 64, 16), (4, 1, 128, 8)])
def test_what_is_not_finite(way, n_q, n_kv, d, page):
    few.test_values_that_are_not_finite(torch.bfloat16, n_q, n_kv, d, page, 40)
    few.test_keys_that_are_not_finite(torch.bfloat16, n_q, n_kv, d, page, 40)


def test_again_and_captured(way):
    few.test_same_bits_every_time_and_on_another_stream(torch.bfloat16, 40)
    few.test_captured_and_replayed(40)
