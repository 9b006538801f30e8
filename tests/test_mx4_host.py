"""4-bit storage without a GPU: the checks of arguments, the size helpers, the refusals."""
import pytest
import torch

import neuzip
from neuzip_b200 import _lib, layerwise
from neuzip_b200.mx4 import _Entry, _stack
from tests import mx4ref


def manager_with(shape, name="w"):
    """A manager that holds `shape` on the CPU: enough for every check that precedes a launch."""
    m = neuzip.MX4Manager()
    stack = _stack(shape)
    L = _lib.load()
    m._be._cache[name] = _Entry(torch.Size(shape), torch.bfloat16, *stack,
                                torch.zeros(int(L.nz_mx4_bytes(*stack)), dtype=torch.uint8), set())
    m.meta_dict[name] = torch.Size(shape)
    return m


def test_names():
    assert issubclass(neuzip.MX4Manager, neuzip.Manager)
    assert "MX4Manager" in neuzip.__all__ and neuzip.nn.Experts


@pytest.mark.parametrize("shape,stack,tiles,blocks,steps", [
    ((4096, 4096), (1, 4096, 4096), 32, 128, 16),
    ((1, 1), (1, 1, 1), 1, 1, 1),
    ((129, 257), (1, 129, 257), 2, 9, 2),
    ((3, 5, 33), (3, 5, 33), 3, 2, 1),
    ((2, 3, 4, 64), (1, 24, 64), 1, 2, 1),
    ((), (1, 1, 1), 1, 1, 1),
    ((0, 64), (1, 0, 64), 0, 2, 1),
    ((7,), (1, 1, 7), 1, 1, 1),
])
def test_sizes(shape, stack, tiles, blocks, steps):
    # a tile of 128 rows: 16 bytes a row and block, a kilobyte of scales for every 256 columns
    assert _stack(shape) == stack
    assert _lib.load().nz_mx4_bytes(*stack) == tiles * (blocks * 2048 + steps * 1024)


def test_reference_rounds_to_the_nearest_code():
    # block maximum 6 -> scale 1: ties go to the even code, everything above 6 saturates
    v = torch.tensor([[0, .25, .26, .75, 1.25, 1.75, 2.5, 3.5, 5, 5.01, -.25, -5, 7.9, 6, -0.74, 2.49]])
    want = [0, 0, .5, 1, 1, 2, 2, 4, 4, 6, 0, -4, 6, 6, -.5, 2]
    assert mx4ref.quantize(v)[0].tolist() == want
    assert mx4ref.quantize(torch.tensor([[8.0, 1.0, 0.5]]))[0].tolist() == [8.0, 1.0, 0.0]
    assert torch.isnan(mx4ref.quantize(torch.tensor([[1.0, float("inf")]]))).all()


@pytest.mark.parametrize("x,error", [
    (torch.zeros(2, 64), RuntimeError),                                   # fp32
    (torch.zeros(2, 63, dtype=torch.bfloat16), ValueError),               # width
    (torch.zeros((), dtype=torch.bfloat16), ValueError),                  # no dimension
    (torch.zeros(2, 64, dtype=torch.bfloat16, device="meta"), ValueError),   # another device
    (torch.zeros(2, 64, dtype=torch.bfloat16, requires_grad=True), RuntimeError),
])
def test_linear_refuses(x, error):
    m = manager_with((32, 64))
    with pytest.raises(error):
        m.linear("w", x)


@pytest.mark.parametrize("bias", [torch.zeros(32), torch.zeros(31, dtype=torch.bfloat16),
                                  torch.zeros(32, dtype=torch.float16),
                                  torch.zeros(32, dtype=torch.bfloat16, device="meta")])
def test_linear_refuses_a_bias(bias):
    with pytest.raises(ValueError):
        manager_with((32, 64)).linear("w", torch.zeros(2, 64, dtype=torch.bfloat16), bias)


def test_linear_needs_a_matrix():
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    for shape in ((4, 32, 64), (64,), (2, 2, 4, 64)):
        with pytest.raises(ValueError):
            manager_with(shape).linear("w", x)
    with pytest.raises(RuntimeError, match="Data not found"):
        m = manager_with((32, 64))
        m.meta_dict["v"] = torch.Size((32, 64))
        m.linear("v", x)


def test_grouped_linear_refuses():
    m = manager_with((4, 32, 64))
    x = torch.zeros(5, 64, dtype=torch.bfloat16)
    ids = torch.zeros(5, 2, dtype=torch.int64)
    with pytest.raises(ValueError, match="stack"):
        manager_with((32, 64)).grouped_linear("w", x, ids)
    for bad in (ids.float(), ids.bool(), ids.to(torch.complex64)):
        with pytest.raises(TypeError):
            m.grouped_linear("w", x, bad)
    for shape in ((4, 2), (5, 2, 2), ()):
        with pytest.raises(ValueError):
            m.grouped_linear("w", x, torch.zeros(shape, dtype=torch.int64))
    with pytest.raises(ValueError):
        m.grouped_linear("w", x, ids.to("meta"))
    with pytest.raises(ValueError):
        m.grouped_linear("w", x, ids, torch.zeros(32, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="gradient"):
        m.grouped_linear("w", x.requires_grad_(), ids)


def test_empty_calls_launch_nothing():
    m = manager_with((4, 32, 64))
    y = m.grouped_linear("w", torch.zeros(0, 64, dtype=torch.bfloat16), torch.zeros(0, 2, dtype=torch.int64))
    assert y.shape == (0, 2, 32)
    y = m.grouped_linear("w", torch.zeros(5, 64, dtype=torch.bfloat16), torch.zeros(5, 0, dtype=torch.int64))
    assert y.shape == (5, 0, 32)
    y = manager_with((32, 64)).linear("w", torch.zeros(3, 0, 64, dtype=torch.bfloat16))
    assert y.shape == (3, 0, 32)


def test_write_refuses_other_types():
    for dtype in (torch.float32, torch.float64, torch.int8):
        with pytest.raises(RuntimeError, match="Unsupported data type"):
            neuzip.MX4Manager().write(torch.zeros(4, 4, dtype=dtype))


def test_split_and_layerwise_are_refused():
    m = neuzip.MX4Manager()
    with pytest.raises(NotImplementedError):
        m.split(torch.zeros(4, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="decode ahead"):
        layerwise.attach(torch.nn.Sequential(), m)


def test_experts_refuses():
    w = torch.zeros(4, 8, 16, dtype=torch.bfloat16)
    with pytest.raises(TypeError):
        neuzip.nn.Experts(neuzip.Manager(algorithm=neuzip.Algorithm.dummy), w)
    with pytest.raises(ValueError):
        neuzip.nn.Experts(neuzip.MX4Manager(), w[0])
    with pytest.raises(ValueError):
        neuzip.nn.Experts(neuzip.MX4Manager(), w, torch.zeros(4, 7))


def test_import_refuses_what_does_not_fit():
    m = neuzip.MX4Manager()
    blob = {"format": "MXFP4", "dtype": "bfloat16", "shape": (4, 64), "stack": (1, 4, 64),
            "packed": torch.zeros(2 * 2048 + 1024, dtype=torch.uint8)}
    for change in ({"format": "NZR1"}, {"dtype": "float32"}, {"shape": (4, 65)},
                   {"packed": torch.zeros(5119, dtype=torch.uint8)}, {"packed": torch.zeros(5120)}):
        with pytest.raises(ValueError):
            m.import_entry({**blob, **change}, "w")


def test_library_refuses_bad_arguments():
    L = _lib.load()
    assert L.nz_mx4_quantize(0, 2, 1, 1, 1, 0, 0) == _lib.NZ_E_ARG
    assert L.nz_mx4_quantize(0, 0, 1, 1, 1, 0, 0) == _lib.NZ_E_ARG
    assert L.nz_mx4_quantize(0, 0, 1, 1 << 31, 1, 0, 0) == _lib.NZ_E_ARG
    assert L.nz_mx4_quantize(16, 0, 1, 1, 1, 8, 0) == _lib.NZ_E_ARG
    assert L.nz_mx4_dequantize(0, 1, 1, 1, 7, 0, 0) == _lib.NZ_E_ARG
    assert L.nz_mx4_dequantize(16, 1, 1, 1, 0, 0, 0) == _lib.NZ_E_ARG
    assert L.nz_mx4_gather_rows(16, 1, 1, 1, 0, 0, 1, 16, 0, 0) == _lib.NZ_E_ARG
    # product: stored bytes, matrices, rows, cols, dtype, x, stride, n_rows, per_input, experts, bias,
    # y, workspace, bytes, status, stream
    good = [16, 1, 4096, 4096, 0, 16, 4096, 40000, 1, 0, 0, 16, 256, 1 << 32, 16, 0]
    assert L.nz_mx4_linear_workspace_bytes(1, 4096, 4096, 40000, 0) > 0
    for at, value in ((0, 0), (0, 8), (2, 1 << 31), (4, 3), (5, 0), (5, 1), (6, 4095), (8, 0), (8, 7), (1, 2),
                      (11, 0), (12, 16), (7, 1 << 31), (10, 1), (9, 4)):
        bad = list(good)
        bad[at] = value
        assert L.nz_mx4_linear(*bad) == _lib.NZ_E_ARG, (at, value)
    for at in (12, 13):
        bad = list(good)
        bad[at] = 0
        assert L.nz_mx4_linear(*bad) == _lib.NZ_E_CAPACITY
    assert L.nz_mx4_linear(*([0, 0, 8, 64] + [0] * 12)) == _lib.NZ_OK      # no rows: nothing to do
