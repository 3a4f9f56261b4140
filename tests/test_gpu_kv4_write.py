"""Rows rounded to 4 bits into the paged cache and pages read back: to the last bit what the definition gives."""
import math

import pytest
import torch

from plain import kv4_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _rows(T, width, kind, g):
    x = torch.randn(T, width, generator=g)
    if kind == "spread":                                    # groups of very different sizes, some below and some above what a scale can be
        x *= torch.exp2(torch.randint(-24, 24, (T, width // 32), generator=g).float()).repeat_interleave(32, 1)
    elif kind == "ties":                                    # halves of scales that are there, and what lies beside them
        scale = (8 + torch.randint(0, 8, (T, width // 32), generator=g)) * torch.exp2(torch.randint(-14, 8, (T, width // 32), generator=g).float())
        scale = scale.repeat_interleave(32, 1)
        x = (torch.randint(-13, 14, (T, width), generator=g) / 2) * scale
        x[:, ::32] = 7 * scale[:, ::32]
        near = torch.randint(0, 3, (T, width), generator=g)
        x = torch.where(near == 1, torch.nextafter(x, torch.full_like(x, math.inf)), torch.where(near == 2, torch.nextafter(x, torch.full_like(x, -math.inf)), x))
    elif kind == "scales":                                  # largest magnitudes whose seventh lies on the border between two scales, and beside it
        border = (2 * (8 + torch.randint(0, 8, (T, width // 32), generator=g)) + 1) * torch.exp2(torch.randint(-16, 8, (T, width // 32), generator=g).float())
        top = 7 * border
        near = torch.randint(0, 3, top.shape, generator=g)
        top = torch.where(near == 1, torch.nextafter(top, torch.full_like(top, math.inf)), torch.where(near == 2, torch.nextafter(top, torch.zeros_like(top)), top))
        x = (torch.rand(T, width, generator=g) * 2 - 1) * top.repeat_interleave(32, 1)
        x[:, 5::32] = -top
    elif kind == "ends":
        x[0] = 0.0
        x[1 % T] *= 1e30
        x[2 % T] = 7 * 61440.0
        x[3 % T, ::7] = 1e-38
        x[4 % T] *= 2.0 ** -17
    elif kind == "odd":
        x[0, 3], x[1 % T, 40 % width], x[2 % T, -1] = math.inf, math.nan, -math.inf
    return x


def _check(k, v, slots, n_kv, d, page, pages, g):
    from photon_infer_b200.kernels import ops
    caches = [plain.random_pool(pages, n_kv, page, d, g) for _ in range(2)]
    got = [c.to(DEV) for c in caches]
    err = torch.zeros(4, dtype=torch.int32, device=DEV)
    ops.kv4_write(k, v, torch.tensor(slots, dtype=torch.int32, device=DEV), got[0], got[1], n_kv, d, err)
    for cache, mine, x, values in zip(caches, got, (k, v), (False, True)):
        codes, scales = (p.clone() for p in plain.page_parts(cache, page, d))
        host = x.float().cpu().tolist()
        for t, slot in enumerate(slots):
            for h in range(n_kv):
                if 0 <= slot < pages * page:
                    c, b = plain.row_bits(host[t][h * d:(h + 1) * d], values)
                    codes[slot // page, h, slot % page] = torch.tensor(c, dtype=torch.uint8)
                    scales[slot // page, h, slot % page] = torch.tensor(b, dtype=torch.uint8)
        want = torch.cat([codes.flatten(2), scales.flatten(2)], 2)
        assert torch.equal(mine.cpu(), want), (mine.cpu() != want).nonzero()[:5]
    return got, err.tolist()


@pytest.mark.parametrize("kind", ["plain", "spread", "ties", "scales", "ends", "odd"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n_kv,d,page", [(2, 64, 8), (1, 128, 4), (3, 32, 16), (1, 96, 16), (1, 256, 2)])
def test_write(kind, dtype, n_kv, d, page):
    g = torch.Generator().manual_seed(d + page)
    T = 13
    k, v = (_rows(T, n_kv * d, kind, g).to(dtype).to(DEV) for _ in range(2))
    slots = torch.randperm(5 * page, generator=g)[:T].tolist() if 5 * page >= T else list(range(5 * page)) + [-1] * (T - 5 * page)
    _, err = _check(k, v, slots, n_kv, d, page, 5, g)
    assert err[0] == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [1, 2, 33])
@pytest.mark.parametrize("offset", [0, 1, 8])
def test_sections_of_a_row(dtype, T, offset):
    """Keys and values as views of a projection's rows, on 16-byte boundaries or beside them."""
    g = torch.Generator().manual_seed(T)
    n_kv, d = 2, 64
    wide = torch.randn(T, offset + 3 * n_kv * d + 1, generator=g).to(dtype).to(DEV)
    k, v = wide[:, offset:offset + n_kv * d], wide[:, offset + 2 * n_kv * d:offset + 3 * n_kv * d]
    _check(k, v, torch.randperm(64, generator=g)[:T].tolist(), n_kv, d, 16, 4, g)


def test_slots_that_are_not_there():
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(4, 64, generator=g).to(DEV) for _ in range(2))
    _, err = _check(k, v, [5, -1, 3 * 8, 2], 1, 64, 8, 3, g)
    assert err == [2, 2, 24, 24]                            # a slot behind the pool, at token 2
    _, err = _check(k, v, [5, -2, 7, 2], 1, 64, 8, 3, g)
    assert err[:3] == [2, 1, -2]


def test_no_tokens():
    from photon_infer_b200.kernels import ops
    pool = plain.random_pool(2, 1, 8, 64, torch.Generator().manual_seed(0)).to(DEV)
    empty, before = torch.empty(0, 64, device=DEV), pool.clone()
    ops.kv4_write(empty, empty, torch.empty(0, dtype=torch.int32, device=DEV), pool, pool.clone(), 1, 64, None)
    assert torch.equal(pool, before)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n_kv,d,page", [(2, 64, 8), (1, 128, 4), (3, 32, 16), (1, 96, 16), (2, 256, 2), (8, 128, 64)])
def test_unpack(dtype, n_kv, d, page):
    """Any bytes at all: every code and every scale, those that stand for no number among them."""
    from photon_infer_b200.kernels import ops
    g = torch.Generator().manual_seed(page)
    k, v = (torch.randint(0, 256, (6, n_kv, ops.kv4_page_bytes(page, d)), generator=g, dtype=torch.uint8) for _ in range(2))
    pages = [4, 0, 6, 0, 5, -1]
    outs = [torch.full((len(pages), n_kv, page, d), 3.0, dtype=dtype, device=DEV) for _ in range(2)]
    err = torch.zeros(4, dtype=torch.int32, device=DEV)
    ops.kv4_unpack(k.to(DEV), v.to(DEV), torch.tensor(pages, dtype=torch.int32, device=DEV), *outs, err)
    for cache, out, values in zip((k, v), outs, (False, True)):
        want = plain.numbers(cache, page, d, values)
        for i, p in enumerate(pages):
            expect = want[p] if 0 <= p < 6 else torch.full_like(want[0], 3.0)
            assert torch.equal(torch.nan_to_num(out[i].double().cpu(), nan=1e9), torch.nan_to_num(expect, nan=1e9))
    assert err[0].item() == 3


def test_places_behind_31_bits():
    """A pool of more than 2^31 bytes: its last pages."""
    from photon_infer_b200.kernels import ops
    n_kv, d, page = 8, 256, 64
    pages = (1 << 31) // (n_kv * ops.kv4_page_bytes(page, d)) + 3
    k, v = (torch.zeros(pages, n_kv, ops.kv4_page_bytes(page, d), dtype=torch.uint8, device=DEV) for _ in range(2))
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2, n_kv * d, generator=g).to(torch.bfloat16).to(DEV)
    slots = [(pages - 1) * page + 5, (pages - 2) * page]
    ops.kv4_write(x, -x, torch.tensor(slots, dtype=torch.int32, device=DEV), k, v, n_kv, d, None)
    outs = [torch.empty(2, n_kv, page, d, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    ops.kv4_unpack(k, v, torch.tensor([pages - 1, pages - 2], dtype=torch.int32, device=DEV), *outs, None)
    for i, slot in enumerate((5, 0)):
        want = torch.tensor([plain.row_bits(x[i, h * d:(h + 1) * d].float().tolist(), False)[1] for h in range(n_kv)])
        assert torch.equal(k[pages - 1 - i, :, page * d // 2 + slot * 8:page * d // 2 + slot * 8 + 8].cpu().long(), want)
        assert torch.equal(outs[0][i, :, slot], -outs[1][i, :, slot]) and outs[0][i, :, slot].abs().sum() > 0
