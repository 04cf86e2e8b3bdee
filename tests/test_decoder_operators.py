"""What rope, rope_cache_update, route_experts and adapter_matmul refuse: no GPU."""
import ctypes

import pytest
import torch

import mlx_amd
from mlx_amd import _lib

BF16 = torch.bfloat16


def z(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype)


def ints(*shape, dtype=torch.int32):
    return torch.zeros(shape, dtype=dtype)


ROPE = dict(x=z(2, 4, 3, 64), positions=ints(2, 3))


@pytest.mark.parametrize("change, words", (
    (dict(x=z(4, 3, 64)), "4 dimensions"),
    (dict(x=z(2, 4, 3, 64, dtype=torch.float64)), "unsupported type"),
    (dict(positions=None), "positions are needed"),
    (dict(positions=ints(3, 2)), "positions"),
    (dict(positions=ints(3, 2, 3)), "positions"),
    (dict(positions=z(2, 3)), "integers"),
    (dict(dims=63), "dims"),
    (dict(x=z(2, 4, 3, 7), dims=2), "must be even"),
    (dict(dims=0), "dims"),
    (dict(dims=66), "dims"),
    (dict(x=z(2, 4, 3, 512)), "at most 256"),
    (dict(base=0.0), "base"),
    (dict(base=float("inf")), "base"),
    (dict(scale=float("nan")), "scale"),
    (dict(base=10.0, freqs=torch.ones(32)), "Only one"),
    (dict(freqs=torch.ones(31)), "freqs"),
    (dict(freqs=ints(32)), "freqs"),
    (dict(sections=(16, 16)), "positions"),
    (dict(sections=(16, 15), positions=ints(2, 2, 3)), "sections"),
    (dict(sections=(33, -1), positions=ints(2, 2, 3)), "sections"),
    (dict(sections=(8, 8, 8, 4, 4), positions=ints(5, 2, 3)), "sections"),
))
def test_rope_refuses(change, words):
    with pytest.raises(ValueError, match=words):
        mlx_amd.rope(**{**ROPE, **change})


UPDATE = dict(q=z(2, 4, 3, 64), k=z(2, 2, 3, 64), v=z(2, 2, 3, 64), k_pages=z(5, 2, 16, 64),
              v_pages=z(5, 2, 16, 64), block_table=ints(2, 2), lengths=ints(2))


@pytest.mark.parametrize("change, words", (
    (dict(q=z(4, 3, 64)), "4 dimensions"),
    (dict(v=z(2, 2, 4, 64)), "same shape"),
    (dict(q=z(2, 4, 2, 64)), "do not go with"),
    (dict(q=z(1, 4, 3, 64)), "do not go with"),
    (dict(k=z(2, 1, 3, 64), v=z(2, 1, 3, 64)), "do not fit"),
    (dict(q=z(2, 4, 3, 64, dtype=torch.float16)), "one real floating type"),
    (dict(block_table=ints(3, 2)), "block_table"),
    (dict(lengths=ints(2, 1)), "lengths"),
    (dict(k_pages=z(5, 2, 24, 64), v_pages=z(5, 2, 24, 64)), "multiple of 16"),
    (dict(k_pages=z(1, 2, 16, 64).expand(5, 2, 16, 64)), "share memory"),
    (dict(sections=(16, 16)), "sections need positions"),
    (dict(positions=ints(2, 2)), "positions"),
    (dict(dims=65), "dims"),
))
def test_rope_cache_update_refuses(change, words):
    with pytest.raises(ValueError, match=words):
        mlx_amd.rope_cache_update(**{**UPDATE, **change})


ROUTE = dict(logits=z(5, 24), k=4)


@pytest.mark.parametrize("change, words", (
    (dict(logits=z(5, 0)), "experts"),
    (dict(logits=z(5, 1025)), "1024"),
    (dict(logits=ints(5, 24)), "unsupported type"),
    (dict(scoring="relu"), "scoring"),
    (dict(groups=5), "groups"),
    (dict(groups=24), "groups"),
    (dict(groups=0), "groups"),
    (dict(groups=4, top_groups=5), "groups"),
    (dict(groups=4, top_groups=0), "groups"),
    (dict(group_best=3), "group_best"),
    (dict(logits=z(5, 16), groups=16, group_best=2), "group_best"),
    (dict(k=0), "k must be"),
    (dict(k=25), "k must be"),
    (dict(logits=z(5, 64), k=33), "at most 32"),
    (dict(groups=8, top_groups=1), "at most 3"),
    (dict(bias=torch.zeros(23)), "bias"),
    (dict(bias=ints(24)), "bias"),
    (dict(scale=float("inf")), "scale"),
))
def test_route_experts_refuses(change, words):
    with pytest.raises(ValueError, match=words):
        mlx_amd.route_experts(**{**ROUTE, **change})


ADAPT = dict(x=z(2, 3, 32), a=z(4, 8, 32), b=z(4, 48, 8), indices=ints(2))


@pytest.mark.parametrize("change, words", (
    (dict(a=z(8, 32)), "shapes"),
    (dict(a=z(3, 8, 32)), "shapes"),
    (dict(a=z(4, 9, 32)), "shapes"),
    (dict(a=z(4, 257, 32), b=z(4, 48, 257)), "rank 1 to 256"),
    (dict(a=z(1025, 1, 32), b=z(1025, 48, 1)), "1024 adapters"),
    (dict(a=z(4, 0, 32), b=z(4, 48, 0)), "rank 1 to 256"),
    (dict(b=z(4, 0, 8)), "possible"),
    (dict(x=z(2, 3, 31)), "last dimension"),
    (dict(y=z(2, 3, 47)), "y must have"),
    (dict(indices=None), "indices are needed"),
    (dict(indices=ints(3)), "first dimensions"),
    (dict(indices=ints(2, 2)), "first dimensions"),
    (dict(indices=z(2)), "integers"),
    (dict(scale=torch.zeros(3)), "scale"),
    (dict(scale=float("nan")), "scale"),
    (dict(x=z(2, 3, 32, dtype=torch.float64)), "unsupported type"),
))
def test_adapter_matmul_refuses(change, words):
    with pytest.raises(ValueError, match=words):
        mlx_amd.adapter_matmul(**{**ADAPT, **change})


def test_gpu_only():
    for call, args in ((mlx_amd.rope, ROPE), (mlx_amd.rope_cache_update, UPDATE),
                       (mlx_amd.route_experts, ROUTE), (mlx_amd.adapter_matmul, ADAPT)):
        with pytest.raises(RuntimeError, match="GPU only"):
            call(**args)


def test_no_forward_mode_and_no_gradients_through_the_cache():
    import torch.autograd.forward_ad as fwad

    with fwad.dual_level():
        for call, args, name in ((mlx_amd.rope, ROPE, "x"), (mlx_amd.rope_cache_update, UPDATE, "q"),
                                 (mlx_amd.route_experts, ROUTE, "logits"),
                                 (mlx_amd.adapter_matmul, ADAPT, "x")):
            dual = fwad.make_dual(args[name], torch.ones_like(args[name]))
            with pytest.raises(NotImplementedError):
                call(**{**args, name: dual})
    with pytest.raises(NotImplementedError, match="cache"):
        mlx_amd.rope_cache_update(**{**UPDATE, "k": UPDATE["k"].clone().requires_grad_()})
    with pytest.raises(NotImplementedError, match="freqs"):
        mlx_amd.rope(**ROPE, freqs=torch.ones(32, requires_grad=True))
    with pytest.raises(NotImplementedError, match="scale"):
        mlx_amd.adapter_matmul(**ADAPT, scale=torch.ones(4, requires_grad=True))


def test_scales_of_a_single_number():
    """Finite in the 32 bits that the kernels hold, and not what a graph would have to reach."""
    for scale in (1e39, -float("inf"), 10 ** 60):
        with pytest.raises(ValueError, match="finite in 32 bits"):
            mlx_amd.route_experts(**ROUTE, scale=scale)
        with pytest.raises(ValueError, match="finite in 32 bits"):
            mlx_amd.adapter_matmul(**ADAPT, scale=scale)
    scale = torch.tensor(2.0, requires_grad=True)
    with pytest.raises(NotImplementedError, match="scale"):
        mlx_amd.adapter_matmul(**ADAPT, scale=scale)
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU only"):
        mlx_amd.adapter_matmul(**ADAPT, scale=scale)


FACTORS = (
    (mlx_amd.rope, ROPE, dict(freqs=torch.ones(32))),
    (mlx_amd.rope, ROPE, dict(freqs=z(32))),
    (mlx_amd.rope, ROPE, dict(scale=torch.tensor(2.0))),
    (mlx_amd.rope, ROPE, dict(base=torch.tensor(500.0))),
    (mlx_amd.rope_cache_update, UPDATE, dict(freqs=torch.ones(32))),
    (mlx_amd.rope_cache_update, UPDATE, dict(scale=torch.tensor(2.0))),
    (mlx_amd.rope_cache_update, UPDATE, dict(base=torch.tensor(500.0))),
    (mlx_amd.route_experts, ROUTE, dict(scale=torch.tensor(2.0))),
    (mlx_amd.adapter_matmul, ADAPT, dict(scale=torch.tensor(2.0))),
    (mlx_amd.adapter_matmul, ADAPT, dict(scale=torch.ones(4))),
)


@pytest.mark.parametrize("call, args, factor", FACTORS)
def test_gradients_of_factors_are_refused_not_dropped(call, args, factor):
    import torch.autograd.forward_ad as fwad

    (name, value), = factor.items()
    with pytest.raises(RuntimeError, match="GPU only"):
        call(**args, **factor)
    with fwad.dual_level(), pytest.raises(NotImplementedError, match="gradients"):
        call(**args, **{name: fwad.make_dual(value, torch.ones_like(value))})
    leaf = value.clone().requires_grad_()
    with pytest.raises(NotImplementedError, match="gradients"):
        call(**args, **{name: leaf})
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU only"):
        call(**args, **{name: leaf})


def _status(name, *args):
    lib = _lib.load()
    return getattr(lib, name)(*args), lib.mlxrocm_last_error().decode()


def test_the_library_checks_its_arguments():
    one = ctypes.c_void_p(16)  # never dereferenced: the checks come first
    strides = (ctypes.c_int64 * 19)()
    sections = (ctypes.c_int * 4)(8, 8, 8, 8)

    def rope(dims=64, axes=1, base=1e4, x=one, sections=sections, D=64):
        return _status("mlxrocm_rope", x, one, 1, 2, 3, D, strides, one, strides, 0, axes, sections,
                       dims, 0, base, 1.0, None, 0, 2, None)

    assert rope(dims=63)[0] == _lib.INVALID_ARGUMENT
    assert rope(dims=2, D=7)[0] == _lib.INVALID_ARGUMENT
    assert rope(dims=258, D=512)[0] == _lib.INVALID_ARGUMENT
    assert rope(axes=5)[0] == _lib.INVALID_ARGUMENT
    assert rope(axes=3)[0] == _lib.INVALID_ARGUMENT  # 24 of 32 pairs
    assert rope(axes=2, sections=None)[0] == _lib.INVALID_ARGUMENT
    assert rope(base=-1.0)[0] == _lib.INVALID_ARGUMENT
    assert rope(x=None) == (_lib.INVALID_ARGUMENT, "[rope] null pointer")

    def update(page=16, pages=4, lengths=one):
        return _status("mlxrocm_rope_cache_update", one, one, one, one, one, one, one, lengths, 1, 4, 2,
                       3, 64, pages, page, 2, strides, None, None, 0, 1, None, 64, 0, 1e4, 1.0, None, 2,
                       None)

    assert update(page=24)[0] == _lib.INVALID_ARGUMENT
    assert update(pages=-1)[0] == _lib.INVALID_ARGUMENT
    assert update(lengths=None)[0] == _lib.INVALID_ARGUMENT

    def route(rows=1, experts=24, k=4, groups=1, top=1, best=1, logits=one):
        return _status("mlxrocm_route_experts", logits, None, one, one, rows, experts, experts, k, 0,
                       groups, top, best, 1, 1.0, 2, None)[0]

    bad = _lib.INVALID_ARGUMENT
    assert route(experts=1025) == bad and route(k=0) == bad and route(k=25) == bad
    assert route(groups=5) == bad and route(groups=4, top=5) == bad and route(best=3) == bad
    assert route(logits=None) == bad and route(rows=-1) == bad and route(rows=0) == _lib.OK
    assert route(rows=1 << 40) == _lib.UNSUPPORTED

    def adapt(rows=6, n=2, adapters=4, rank=8, x=one, ws=0):
        return _status("mlxrocm_adapter_matmul", x, one, one, one, None, None, one, None, rows, n,
                       adapters, rank, 32, 48, 32, 48, 1.0, 2, one, ws, None)[0]

    assert adapt(rows=5) == bad and adapt(n=0) == bad and adapt(adapters=0) == bad
    assert adapt(rank=257) == bad and adapt(x=None) == bad and adapt() == bad  # no workspace
    assert adapt(rows=0, n=0) == _lib.OK and adapt(rows=1 << 25, n=1) == _lib.UNSUPPORTED
