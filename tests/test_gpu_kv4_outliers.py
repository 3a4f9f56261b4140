"""Values of very different sizes side by side, where the large ones have no weight: what is left is the small ones', to its last bit."""
import math

import pytest
import torch

from plain import kv4_plain as plain
from test_gpu_kv4_attention import Step, near

pytestmark = pytest.mark.gpu


def _place(step, s, key):
    return int(step.table[s, key // step.page]), key % step.page


def _set_scales(step, cache, s, key, byte):
    page, slot = _place(step, s, key)
    groups = step.d // 32
    at = step.page * step.d // 2 + slot * groups
    cache[page, :, at:at + groups] = byte


def _set_codes(step, cache, s, key, code):
    page, slot = _place(step, s, key)
    cache[page, :, slot * step.d // 2:(slot + 1) * step.d // 2] = code | code << 4


@pytest.mark.parametrize("low,high", [(1, 16), (40, 64), (100, 104)])
@pytest.mark.parametrize("large", [150, 200, 247])
@pytest.mark.parametrize("tokens", [1, 2, 8])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_large_values_that_have_no_weight(dtype, d, tokens, large, low, high):
    """Queries are positive and so are the keys, but for those of the large values: their scores lie hundreds below the others'."""
    held = 300
    step = Step([tokens], [held], 4, 2, d, 16, dtype, seed=d + large + low, sharp=1.0)
    step.q = (step.q.float().abs() + 0.5).to(dtype)
    step.v = plain.random_pool(step.pages, 2, 16, d, step.g, low, high)
    for key in range(held):
        _set_codes(step, step.k, 0, key, 9 + key % 2)
        _set_scales(step, step.k, 0, key, 104)                       # 1/4
    for key in (0, 3, 64, 65, 100, 170, 280):
        _set_codes(step, step.k, 0, key, 1)
        _set_scales(step, step.k, 0, key, 168)                       # 64
        _set_scales(step, step.v, 0, key, large)
    got, _ = step.run()
    want, _, off, _ = step.want()
    near(got, want, off)


@pytest.mark.parametrize("d", [64, 128])
def test_large_values_that_other_rows_see(d):
    """The last token's own key has the largest values: the tokens in front of it keep their small results."""
    step = Step([3], [200], 4, 2, d, 16, torch.bfloat16, seed=d)
    step.v = plain.random_pool(step.pages, 2, 16, d, step.g, 1, 16)
    _set_scales(step, step.v, 0, 199, 247)
    got, _ = step.run()
    want, _, off, _ = step.want()
    # Numbers 2 i and 2 i + 1 of a head share a sum over (c0 + 16 c1) times the weights, and the first is what is left of it without the second (16 c1): both sums have the size of 16 times
    # the second's, and a product of 16 keys adds to them with 23 bits.  So the first is off by that part of the second, 2^-20 or so of a group's scale, which stands for half a scale itself.
    k, v = step.rows(0, step.k, False), step.rows(0, step.v, True)
    mass = plain.attention(step.q.double().view(3, 4, d), k, v, 3, 200, 2, d ** -0.5)[3]
    other = mass.view(3, 4, d // 2, 2).flip(-1).reshape(3, 4 * d)
    near(got, want, off + other * 16 * (2 * (200 // 16 + 3)) * 2.0 ** -23)
    near(got[:2], want[:2], off[:2])


def test_one_key_above_many_small_ones_beside_large_values():
    """65,536 keys whose weights are each 2^-17 of the largest one's and together half of its, values of the smallest scale, and among every 16 of them a large value without weight."""
    n, d = 65537, 64
    step = Step([1], [n], 1, 1, d, 16, torch.bfloat16, seed=53)
    for cache, code, byte in ((step.k, 8, 40), (step.v, 9, 1)):
        cache[:, :, :16 * 32] = code | code << 4
        cache[:, :, 16 * 32:] = byte
    large = 0
    for page in range(step.table.shape[1] - 2):                       # the first key of every page but the last
        p = int(step.table[0, page])
        step.k[p, 0, 0] = 0x01 | 0x80                                 # number 0 of the head: -7 scales
        step.k[p, 0, 16 * 32] = 160                                   # 32
        step.v[p, 0, 16 * 32:16 * 32 + 2] = 200
        large += 1
    page, slot = int(step.table[0, 30001 // 16]), 30001 % 16
    step.k[page, 0, slot * 32] = 0x0F | 0x80
    step.k[page, 0, 16 * 32 + slot * 2] = 120                         # 1.0
    step.v[page, 0, slot * 32:slot * 32 + 32] = 7 | 7 << 4            # -1 scale
    step.q[:] = 0
    step.q[0, 0] = 1.6875                                             # a score of 11.8125 in front of zeros; -378 for the large values
    got, _ = step.run(scale=1.0)
    top, scale = math.exp(7 * 1.6875), plain.scale_of(1)
    want = scale * ((n - 1 - large) - top) / ((n - 1 - large) + top)
    # a weight and its product with the scale are rounded to 11 bits each, the result to 8
    mass = scale
    assert bool(((got.double().cpu() - want).abs() <= abs(want) * 2.0 ** -8 + mass * 2.0 ** -9).all()), (got.double().cpu()[0, :4].tolist(), want)
