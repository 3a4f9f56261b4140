"""Caches in 4 bits, weights of keys and eviction: which calls are refused, and with what; checked without a GPU."""
import pytest
import torch

from photon_infer_b200.errors import ErrorCode, PhotonError
from photon_infer_b200.kernels import ops
from plain import kv4_plain as plain


@pytest.fixture(autouse=True)
def host(monkeypatch):
    """Tensors of the host go through the checks; a call that passes them all must not reach a kernel."""
    def reached(*a, **k):
        raise AssertionError("a kernel was reached")
    monkeypatch.setattr(ops, "_on_device", lambda what, *t: 0)
    monkeypatch.setattr(ops, "_cuda", lambda *t: None)
    monkeypatch.setattr(ops, "_plain_fn", reached)
    monkeypatch.setattr(ops, "sm_count", lambda device: 148)


def _refused(code, call, *args, **kwargs):
    with pytest.raises(PhotonError) as e:
        call(*args, **kwargs)
    assert e.value.code == code, e.value


def _ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def _pool(pages=4, n_kv=2, page=16, d=64):
    return torch.zeros(pages, n_kv, ops.kv4_page_bytes(page, d), dtype=torch.uint8)


def test_page_bytes():
    assert ops.kv4_page_bytes(16, 64) == 16 * 34 and ops.kv4_page_bytes(16, 128) == 16 * 68 and ops.kv4_page_bytes(2, 256) == 2 * 136
    for page, d in ((16, 48), (16, 0), (16, 288), (4, 64), (0, 64), (8, 96), (15, 128), (-8, 64)):
        _refused(ErrorCode.UNSUPPORTED_SIZE, ops.kv4_page_bytes, page, d)
        assert not ops.kv4_supported(page, d)


def test_tensors_of_the_host_are_refused(monkeypatch):
    monkeypatch.undo()
    _refused(ErrorCode.INVALID_ARGUMENT, ops.kv4_write, torch.zeros(3, 128), torch.zeros(3, 128), _ints(3), _pool(), _pool(), **WRITE)
    _refused(ErrorCode.INVALID_ARGUMENT, ops.kv4_attention, **_attention())
    _refused(ErrorCode.INVALID_ARGUMENT, ops.key_weights, **_weigh())
    _refused(ErrorCode.INVALID_ARGUMENT, ops.cache_evict, **_evict())


def test_tensors_of_another_device_are_refused(monkeypatch):
    """A kernel runs on the current device's stream."""
    monkeypatch.undo()

    class Elsewhere:
        is_cuda = True

        def __init__(self, index):
            self.index = index

        def get_device(self):
            return self.index
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1, raising=False)
    ops._on_device("it", Elsewhere(1), None, Elsewhere(1))
    _refused(ErrorCode.INVALID_ARGUMENT, ops._on_device, "it", Elsewhere(1), Elsewhere(0))


WRITE = dict(n_kv=2, head_dim=64, err=None)


def test_write():
    k, v, at = torch.zeros(3, 128), torch.zeros(3, 128), _ints(3)
    for bad in (dict(k=torch.zeros(3, 64)), dict(k=torch.zeros(2, 128)), dict(v=torch.zeros(3, 128, dtype=torch.bfloat16)), dict(v=torch.zeros(128, 3).t()),
                dict(v_cache=_pool(pages=5)), dict(k_cache=_pool(n_kv=1)), dict(k_cache=torch.zeros(4, 2, 33, dtype=torch.uint8)),
                dict(k_cache=_pool().float()), dict(k_cache=_pool(pages=8)[::2])):
        _refused(ErrorCode.SHAPE_MISMATCH, ops.kv4_write, **{**dict(k=k, v=v, slot_mapping=at, k_cache=_pool(), v_cache=_pool()), **bad}, **WRITE)
    _refused(ErrorCode.INVALID_ARGUMENT, ops.kv4_write, k, v, at.long(), _pool(), _pool(), **WRITE)
    _refused(ErrorCode.INVALID_ARGUMENT, ops.kv4_write, k.half(), v.half(), at, _pool(), _pool(), **WRITE)
    _refused(ErrorCode.UNSUPPORTED_SIZE, ops.kv4_write, torch.zeros(3, 96), torch.zeros(3, 96), at, _pool(), _pool(), n_kv=2, head_dim=48, err=None)
    odd = torch.zeros(_pool().numel() + 8, dtype=torch.uint8)
    odd = odd[(8 - odd.data_ptr()) % 16:][:_pool().numel()].view_as(_pool())
    if odd.data_ptr() % 16:
        _refused(ErrorCode.INVALID_ARGUMENT, ops.kv4_write, k, v, at, odd, _pool(), **WRITE)
    with pytest.raises(AssertionError, match="reached"):
        ops.kv4_write(k, v, at, _pool(), _pool(), **WRITE)


def test_unpack():
    good = lambda dtype=torch.float32: torch.zeros(2, 2, 16, 64, dtype=dtype)       # noqa: E731
    for bad in (dict(k_out=torch.zeros(3, 2, 16, 64)), dict(v_out=good(torch.bfloat16)), dict(k_out=torch.zeros(2, 2, 8, 64), v_out=torch.zeros(2, 2, 8, 64)),
                dict(v_cache=_pool(pages=3)), dict(k_out=torch.zeros(2, 16, 2, 64).transpose(1, 2))):
        _refused(ErrorCode.SHAPE_MISMATCH, ops.kv4_unpack, **{**dict(k_cache=_pool(), v_cache=_pool(), pages=_ints(2), k_out=good(), v_out=good(), err=None), **bad})
    _refused(ErrorCode.INVALID_ARGUMENT, ops.kv4_unpack, _pool(), _pool(), _ints(2).long(), good(), good(), None)
    _refused(ErrorCode.INVALID_ARGUMENT, ops.kv4_unpack, _pool(), _pool(), _ints(2), good(torch.float16), good(torch.float16), None)


def _attention(**change):
    a = dict(q=torch.zeros(3, 256), out=torch.zeros(3, 256), k_cache=_pool(), v_cache=_pool(), block_table=_ints(2, 4), cu_tokens=_ints(3), context_lens=_ints(2),
             num_seqs=2, max_tokens_per_seq=2, max_keys=40, n_q=4, n_kv=2, head_dim=64, window=None, scale=0.125, err=None)
    a.update(change)
    return a


def test_attention():
    shapes = [dict(q=torch.zeros(3, 192)), dict(out=torch.zeros(2, 256)), dict(out=torch.zeros(3, 256, dtype=torch.bfloat16)), dict(out=torch.zeros(1, 256).expand(3, 256)),
              dict(q=torch.zeros(256, 3).t()), dict(v_cache=_pool(pages=3)), dict(k_cache=_pool(n_kv=1)), dict(num_seqs=3), dict(block_table=_ints(1, 4)),
              dict(context_lens=_ints(1)), dict(block_table=_ints(8)), dict(sink=torch.zeros(2)), dict(lse=torch.zeros(3, 2)), dict(lse=torch.zeros(3, 4).double())]
    for bad in shapes:
        _refused(ErrorCode.SHAPE_MISMATCH, ops.kv4_attention, **_attention(**bad))
    for bad in (dict(cu_tokens=_ints(3).long()), dict(block_table=_ints(4, 2).t()), dict(scale=0.0), dict(scale=float("nan")), dict(softcap=-1.0), dict(window=-1)):
        _refused(ErrorCode.INVALID_ARGUMENT, ops.kv4_attention, **_attention(**bad))
    for bad in (dict(n_q=3), dict(n_kv=0), dict(head_dim=48, q=torch.zeros(3, 192), out=torch.zeros(3, 192))):
        _refused(ErrorCode.UNSUPPORTED_SIZE, ops.kv4_attention, **_attention(**bad))
    _refused(ErrorCode.INVALID_ARGUMENT, ops.kv4_attention, **_attention(q=torch.zeros(3, 256).half(), out=torch.zeros(3, 256).half()))
    ops.kv4_attention(**_attention(num_seqs=0))                       # nothing to do, nothing launched
    ops.kv4_attention(**_attention(q=torch.zeros(0, 256), out=torch.zeros(0, 256)))
    with pytest.raises(AssertionError, match="reached"):
        ops.kv4_attention(**_attention())


def _weigh(**change):
    a = {k: v for k, v in _attention().items() if k not in ("out", "v_cache")} | dict(weights=torch.zeros(4, 2, 16))
    a.update(change)
    return a


def test_key_weights():
    for bad in (dict(q=torch.zeros(3, 192)), dict(weights=torch.zeros(4, 2, 8)), dict(weights=torch.zeros(4, 2, 16).double()), dict(k_cache=torch.zeros(4, 2, 16, 32)),
                dict(k_cache=torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)), dict(held=_ints(1)), dict(lse=torch.zeros(4)), dict(num_seqs=3), dict(weights=torch.zeros(8, 2, 16)[::2])):
        _refused(ErrorCode.SHAPE_MISMATCH, ops.key_weights, **_weigh(**bad))
    for bad in (dict(held=_ints(2).long()), dict(scale=-1.0), dict(softcap=-2.0), dict(window=-3)):
        _refused(ErrorCode.INVALID_ARGUMENT, ops.key_weights, **_weigh(**bad))
    for bad in (dict(n_q=3), dict(head_dim=12, k_cache=torch.zeros(4, 2, 16, 12), q=torch.zeros(3, 48))):
        _refused(ErrorCode.UNSUPPORTED_SIZE, ops.key_weights, **_weigh(**bad))
    for good in ({}, dict(k_cache=torch.zeros(4, 2, 16, 64))):
        with pytest.raises(AssertionError, match="reached"):
            ops.key_weights(**_weigh(**good))


def _evict(**change):
    a = dict(kv=torch.zeros(3, 2, 4, 2, 16, 64), weights=torch.zeros(3, 4, 2, 16), block_table=_ints(2, 4), context_lens=_ints(2), new_lens=_ints(2), num_seqs=2, max_keys=40,
             keep=8, keep_first=2, keep_last=2, err=None)
    a.update(change)
    return a


def test_evict():
    lens = _ints(4)
    for bad in (dict(kv=torch.zeros(3, 2, 4, 2, 8, 64)), dict(kv=torch.zeros(2, 2, 4, 2, 16, 64)), dict(kv=torch.zeros(3, 2, 4, 2, 16 * 64)), dict(weights=torch.zeros(3, 4, 2, 16).double()),
                dict(kv=torch.zeros(3, 2, 4, 2, 100, dtype=torch.uint8)), dict(kv=torch.zeros(3, 2, 4, 2, 33 * 16, dtype=torch.uint8)), dict(num_seqs=3), dict(new_lens=_ints(1)),
                dict(kept=_ints(3, 2, 2, 7)), dict(kv=torch.zeros(3, 2, 8, 2, 16, 64)[:, :, ::2])):
        _refused(ErrorCode.SHAPE_MISMATCH, ops.cache_evict, **_evict(**bad))
    for bad in (dict(keep=-1), dict(keep_first=-1), dict(keep_last=-1), dict(context_lens=lens[:2], new_lens=lens[:2]), dict(context_lens=lens[:2], new_lens=lens[1:3]),
                dict(context_lens=_ints(2).long()), dict(kv=torch.zeros(3, 2, 4, 2, 16, 64).half())):
        _refused(ErrorCode.INVALID_ARGUMENT, ops.cache_evict, **_evict(**bad))
    _refused(ErrorCode.UNSUPPORTED_SIZE, ops.cache_evict, **_evict(kv=torch.zeros(3, 2, 4, 2, 16, 6)))
    with pytest.raises(AssertionError, match="reached"):
        ops.cache_evict(**_evict(context_lens=lens[:2], new_lens=lens[2:]))
    with pytest.raises(AssertionError, match="reached"):
        ops.cache_evict(**_evict(kv=torch.zeros(3, 2, 4, 2, ops.kv4_page_bytes(16, 64), dtype=torch.uint8)))


def test_structures_are_the_header_s(tmp_path):
    """The packed calls are as long as the C structures."""
    import os
    import shutil
    import subprocess

    from photon_infer_b200.csrc.build import INCLUDE_DIR, find_nvcc
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    names = ("kv4_write", "kv4_unpack", "kv4_attention", "key_weights", "evict")
    src = tmp_path / "sizes.c"
    src.write_text("#include <stdio.h>\n#include <photon/kernels.h>\nint main(void) {\n" + "".join(f'  printf("%zu ", sizeof(photon_{n}_call));\n' for n in names) + "  return 0;\n}\n")
    cuda = os.path.dirname(os.path.dirname(find_nvcc()))
    subprocess.run([cc, "-I", INCLUDE_DIR, "-I", os.path.join(cuda, "include"), str(src), "-o", str(tmp_path / "sizes")], check=True)
    sizes = [int(x) for x in subprocess.run([str(tmp_path / "sizes")], capture_output=True, text=True, check=True).stdout.split()]
    assert sizes == [getattr(ops, f"_{n.upper()}_CALL").size for n in names]


def test_plain_format_by_hand():
    codes, byte = plain.group_bits([7.0] + [0.5, 1.5, -2.5, 3.4999] + [0.0] * 27)
    assert plain.scale_of(byte) == 1.0 and codes[:5] == [15, 8, 10, 6, 11] and codes[5:] == [8] * 27
    assert plain.group_bits([float("inf")] + [1.0] * 31) == ([8] * 32, 255)
    assert plain.group_bits([0.0] * 32) == ([8] * 32, 0)
    assert plain.scale_of(plain.group_bits([1e9] + [0.0] * 31)[1]) == 61440.0
    assert sorted(plain.place(128, False)) == list(range(128)) == sorted(plain.place(128, True))
    assert plain.kept_places([5, 1, float("nan"), 1, 2, 0, 9], 7, 4, 1, 1) == [0, 2, 4, 6]
    assert plain.kept_places([0, 1, 1, 1, 1, 0], 6, 3, 0, 1) == [1, 2, 5]
    assert plain.kept_places([0.0] * 6, 6, 3, 2, 4) == [0, 1, 5]
