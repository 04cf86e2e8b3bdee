"""What attention, its cache and verify_draft refuse, and which kernels they launch: no GPU."""
import ctypes

import pytest
import torch

import mlx_amd
from mlx_amd import _lib

BF16 = torch.bfloat16


def z(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype)


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


GOOD = dict(q=z(2, 4, 3, 64), k=z(2, 2, 5, 64), v=z(2, 2, 5, 64), scale=1.0)


@pytest.mark.parametrize("change, words", (
    (dict(q=z(4, 3, 64)), "4 dimensions"),
    (dict(v=z(2, 2, 4, 64)), "same shape"),
    (dict(q=z(2, 4, 3, 72)), "last dimensions"),
    (dict(q=z(2, 3, 3, 64)), "cannot share"),
    (dict(q=z(3, 4, 3, 64)), "batch size"),
    (dict(q=z(2, 4, 3, 60), k=z(2, 2, 5, 60), v=z(2, 2, 5, 60)), "multiple of 8"),
    (dict(q=z(2, 4, 3, 264), k=z(2, 2, 5, 264), v=z(2, 2, 5, 264)), "up to 256"),
    (dict(window=0), "window"),
    (dict(keep=-1), "keep"),
    (dict(scale=float("nan")), "finite"),
    (dict(lengths=ints(3)), "lengths"),
    (dict(lengths=z(2)), "integers"),
    (dict(q=z(2, 4, 3, 64, dtype=torch.float64)), "unsupported type"),
))
def test_window_attention_refuses(change, words):
    with pytest.raises(ValueError, match=words):
        mlx_amd.window_attention(**{**GOOD, **change})


PAGED = dict(q=z(2, 4, 3, 64), k_pages=z(5, 2, 16, 64), v_pages=z(5, 2, 16, 64),
             block_table=ints(2, 2), lengths=ints(2), scale=1.0)


@pytest.mark.parametrize("change, words", (
    (dict(k_pages=z(5, 2, 8, 64), v_pages=z(5, 2, 8, 64)), "multiple of 16"),
    (dict(v_pages=z(5, 2, 32, 64)), "same shape"),
    (dict(block_table=ints(3, 2)), "block_table"),
    (dict(block_table=ints(2)), "block_table"),
    (dict(block_table=z(2, 2)), "integers"),
    (dict(lengths=ints(2, 1)), "lengths"),
    (dict(q=z(2, 4, 3, 64, dtype=torch.float16)), "one real floating type"),
    (dict(window=-1), "window"),
))
def test_paged_attention_refuses(change, words):
    with pytest.raises(ValueError, match=words):
        mlx_amd.paged_attention(**{**PAGED, **change})


def test_gpu_only():
    with pytest.raises(RuntimeError, match="GPU only"):
        mlx_amd.window_attention(**GOOD)
    with pytest.raises(RuntimeError, match="GPU only"):
        mlx_amd.paged_attention(**PAGED)
    with pytest.raises(RuntimeError, match="GPU only"):
        mlx_amd.paged_cache_update(z(2, 2, 1, 64), z(2, 2, 1, 64), PAGED["k_pages"],
                                   PAGED["v_pages"], ints(2, 2), ints(2))
    with pytest.raises(RuntimeError, match="GPU only"):
        mlx_amd.verify_draft(ints(2, 3), z(2, 4, 9), z(2, 3, 9), torch.zeros(2, 3), torch.zeros(2))


@pytest.mark.parametrize("change, words", (
    (dict(draft=ints(2)), "2 dimensions"),
    (dict(target=z(2, 3, 9)), "target_probs"),
    (dict(probs=z(2, 3, 8)), "draft_probs"),
    (dict(probs=z(2, 3, 9, dtype=torch.float32)), "one real floating type"),
    (dict(target=z(2, 4, 0), probs=None), "empty"),
    (dict(accept=torch.zeros(2, 4)), "accept_uniform"),
    (dict(sample=torch.zeros(2, dtype=torch.float64)), "sample_uniform"),
    (dict(draft=torch.zeros(2, 3)), "integers"),
))
def test_verify_draft_refuses(change, words):
    args = {**dict(draft=ints(2, 3), target=z(2, 4, 9), probs=z(2, 3, 9),
                   accept=torch.zeros(2, 3), sample=torch.zeros(2)), **change}
    with pytest.raises(ValueError, match=words):
        mlx_amd.verify_draft(*args.values())


def test_the_abi_refuses():
    lib = _lib.load()
    one = ctypes.c_void_p(16)  # never read: the checks come first
    s = (ctypes.c_int64 * 24)(*[64] * 24)
    odd = (ctypes.c_int64 * 24)(*[63] * 24)
    bad, unsupported = _lib.INVALID_ARGUMENT, _lib.UNSUPPORTED

    def window(q=one, Hq=4, D=64, strides=s, scale=1.0, window=9, keep=0, dtype=2, keys=70):  # noqa: E501
        return lib.mlxrocm_window_attention(q, one, one, one, None, None, 2, Hq, 2, 3, keys, D,
                                            strides, scale, window, keep, dtype, None, 0, None)

    assert window(q=None) == bad and b"null pointer: q" in lib.mlxrocm_last_error()
    assert window(D=60) == window(D=0) == window(D=264) == window(Hq=3) == bad
    assert window(window=0) == window(keep=-1) == window(dtype=3) == bad
    assert window(scale=float("inf")) == window(strides=None) == bad
    assert window(strides=odd) == window(q=ctypes.c_void_p(8)) == unsupported
    assert window(keys=1 << 20, window=1 << 30) == bad and b"workspace" in lib.mlxrocm_last_error()
    assert window(keys=-1) == bad
    assert lib.mlxrocm_window_attention_workspace_size(2, 3, 2, 3, 70, 64, 9, 0, 2) == 0

    def paged(page=16, width=4, table=one, lengths=one):
        return lib.mlxrocm_paged_attention(one, one, one, table, lengths, one, 2, 4, 2, 3, 64, 9,
                                           page, width, s, 1.0, 9, 0, 2, None, 0, None)

    assert paged(page=0) == paged(page=24) == paged(table=None) == paged(lengths=None) == bad
    assert paged(width=1 << 28) == unsupported
    update = lambda page=16, D=64, v=one: lib.mlxrocm_paged_cache_update(  # noqa: E731
        one, v, one, one, one, one, 2, 2, 3, D, 9, page, 4, s, 2, None)
    assert update(page=8) == update(D=60) == update(v=None) == bad
    verify = lambda V=100, K=3, target=one, size=1 << 20: lib.mlxrocm_verify_draft(  # noqa: E731
        one, target, None, one, one, None, one, one, 2, K, V, s, 2, one, size, None)
    assert verify(V=0) == verify(K=-1) == verify(target=None) == verify(size=0) == bad
    assert verify(V=(1 << 22) + 1) == unsupported


def test_which_kernels_run():
    plan = lambda *a, **k: _lib.attention_plan(*a, **k)[1]  # noqa: E731
    assert plan(64, 32, 8, 1, 100, 128) == "attention_few(dim=128,rows=16,splits=1)"
    assert plan(64, 32, 8, 1, 100, 80).startswith("attention_few(dim=128,")
    assert plan(64, 32, 8, 5, 100, 64).startswith("attention_few(dim=64,rows=32,")
    assert plan(1, 32, 8, 1, 8192, 128).endswith("+attention_join")
    assert plan(1, 32, 8, 4096, 4096, 80) == "attention_rows(dim=96,splits=1)"
    assert plan(1, 32, 8, 128, 32768, 256).startswith("attention_rows(dim=256,splits=")
    # a short window leaves nothing to split
    assert plan(1, 32, 8, 1, 8192, 128, window=128) == "attention_few(dim=128,rows=16,splits=1)"
