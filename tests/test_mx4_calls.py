"""4-bit storage without a GPU: which calls the products take and which they refuse, beyond types and sizes."""
import pytest
import torch

import neuzip
from tests.test_mx4_host import manager_with

BF16 = torch.bfloat16


class Launched(Exception):
    pass


@pytest.fixture
def at_launch(monkeypatch):
    """A product that is let through ends where its kernels would be launched."""
    from neuzip_b200.mx4 import MX4Backend
    calls = []

    def launch(self, entry, x, n_rows, per_input, ids, bias, y):
        calls.append((x, bias, y))
        return y.zero_()
    monkeypatch.setattr(MX4Backend, "_launch", launch)
    return calls


def test_a_bias_may_need_a_gradient(at_launch):
    m = manager_with((32, 64))
    x, bias = torch.zeros(2, 3, 64, dtype=BF16), torch.zeros(32, dtype=BF16, requires_grad=True)
    y = m.linear("w", x, bias)
    assert y.requires_grad and y.shape == (2, 3, 32)
    y.backward(torch.ones_like(y))
    assert torch.equal(bias.grad, torch.full((32,), 6, dtype=BF16))
    with torch.no_grad():
        assert not m.linear("w", x, bias).requires_grad
    with pytest.raises(RuntimeError, match="nn.Linear"):
        m.linear("w", x.clone().requires_grad_(), bias)


def test_the_bias_of_a_stack_has_no_gradient(at_launch):
    m = manager_with((4, 32, 64))
    x, ids = torch.zeros(5, 64, dtype=BF16), torch.zeros(5, 2, dtype=torch.int64)
    bias = torch.zeros(4, 32, dtype=BF16, requires_grad=True)
    with pytest.raises(RuntimeError, match="gradient for its bias"):
        m.grouped_linear("w", x, ids, bias)
    with torch.no_grad():
        assert m.grouped_linear("w", x, ids, bias).shape == (5, 2, 32)
    assert m.grouped_linear("w", x, ids, bias.detach()).shape == (5, 2, 32)


@pytest.fixture
def autocast():
    """Autocast as on a machine with a GPU (torch.autocast switches itself off without one)."""
    on, dtype = torch.is_autocast_enabled("cuda"), torch.get_autocast_dtype("cuda")

    def begin(to):
        torch.set_autocast_enabled("cuda", True)
        torch.set_autocast_dtype("cuda", to)
    yield begin
    torch.set_autocast_enabled("cuda", on)
    torch.set_autocast_dtype("cuda", dtype)


@pytest.mark.parametrize("to", (BF16, torch.float16))
@pytest.mark.parametrize("x_type", (torch.float32, BF16, torch.float16))
@pytest.mark.parametrize("bias_type", (torch.float32, BF16, torch.float16, None))
def test_autocast_takes_inputs_and_bias_to_its_type(at_launch, autocast, to, x_type, bias_type):
    autocast(to)
    ids = torch.zeros(2, 3, dtype=torch.int64)
    bias = [None, None] if bias_type is None else [torch.ones(32, dtype=bias_type), torch.ones(4, 32, dtype=bias_type)]
    assert manager_with((32, 64)).linear("w", torch.ones(2, 64, dtype=x_type), bias[0]).dtype == to
    assert manager_with((4, 32, 64)).grouped_linear("w", torch.ones(2, 64, dtype=x_type), ids, bias[1]).dtype == to
    for x, b, y in at_launch:
        assert x.dtype == to and y.dtype == to and (b is None or b.dtype == to)


def test_autocast_leaves_other_types_refused(at_launch, autocast):
    autocast(BF16)
    for dtype in (torch.float64, torch.int32):
        with pytest.raises(RuntimeError, match="Unsupported data type"):
            manager_with((32, 64)).linear("w", torch.ones(2, 64, dtype=dtype))
    x = torch.ones(2, 64)
    bias = torch.zeros(32, requires_grad=True)
    manager_with((32, 64)).linear("w", x, bias).sum().backward()
    assert bias.grad.dtype == torch.float32 and torch.equal(bias.grad, torch.full((32,), 2.0))


def test_forward_mode_derivatives_are_refused(at_launch):
    from torch.autograd import forward_ad
    m, stack = manager_with((32, 64)), manager_with((4, 32, 64))
    x, bias, ids = torch.zeros(2, 64, dtype=BF16), torch.zeros(32, dtype=BF16), torch.zeros(2, dtype=torch.int64)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: m.linear("w", dual), lambda: stack.grouped_linear("w", dual, ids),
                     lambda: m.linear("w", x, forward_ad.make_dual(bias, torch.ones_like(bias)))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        assert m.linear("w", x, bias).shape == (2, 32)
    assert not forward_ad.unpack_dual(m.linear("w", x, bias)).tangent


def test_the_bias_of_a_stack_has_a_row_for_every_matrix(at_launch):
    m, x, ids = manager_with((4, 32, 64)), torch.zeros(5, 64, dtype=BF16), torch.zeros(5, 2, dtype=torch.int64)
    for shape in ((32, 4), (4 * 32,), (4, 32, 1), (1, 4, 32), (2, 64), (32,)):
        with pytest.raises(ValueError, match="shape"):
            m.grouped_linear("w", x, ids, torch.zeros(shape, dtype=BF16))
    assert m.grouped_linear("w", x, ids, torch.zeros(32, 4, dtype=BF16).t()).shape == (5, 2, 32)
    one = manager_with((32, 64))
    for shape in ((32,), (1, 32), (32, 1)):
        assert one.linear("w", x, torch.zeros(shape, dtype=BF16)).shape == (5, 32)
    for shape in ((33,), (2, 32), (), (0,)):
        with pytest.raises(ValueError, match="shape"):
            one.linear("w", x, torch.zeros(shape, dtype=BF16))


def test_bytes_kept_for_captured_graphs_are_counted_and_released():
    m = manager_with((128, 32))
    size = m.size("w")
    entry = m._be.entry("w")
    assert m.captured_bytes() == 0
    m._be._captured[entry.packed.data_ptr()] = entry.packed            # as a capture does
    assert m.captured_bytes() == 0                                     # the handle holds them too
    m._be._cache["w"] = manager_with((128, 32))._be.entry("w")         # written again
    assert m.captured_bytes() == size and m.total_size() == size
    m._be.erase("w")
    assert m.captured_bytes() == size
    m.release_captured()
    assert m.captured_bytes() == 0 and not m._be._captured


def blob_of(shape=(4, 64), dtype="bfloat16"):
    from neuzip_b200 import _lib
    from neuzip_b200.mx4 import _stack
    stack = _stack(shape)
    return {"format": "MXFP4", "dtype": dtype, "shape": shape, "stack": stack,
            "packed": torch.zeros(int(_lib.load().nz_mx4_bytes(*stack)), dtype=torch.uint8)}


def test_imported_bytes_go_to_the_device_of_what_they_replace(monkeypatch):
    m = manager_with((4, 64))
    be = m._be
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    be.entry("w").device = torch.device("cuda", 1)
    assert be._import_device("w", None) == torch.device("cuda", 1)
    assert be._import_device("w", "cuda:2") == torch.device("cuda", 2)
    assert be._import_device("w", "cuda") == torch.device("cuda", 0)
    assert be._import_device("w", "cpu") == torch.device("cuda", 1)       # stored bytes live on a GPU
    assert be._import_device("new", None) == torch.device("cuda", 0)
    assert be._import_device("new", torch.device("cpu")) == torch.device("cuda", 0)


def test_a_converted_layer_is_loaded_where_it_is_asked_for(monkeypatch):
    from neuzip_b200.mx4 import MX4Backend
    went = []
    monkeypatch.setattr(MX4Backend, "import_entry", lambda self, name, blob, device=None: went.append((name, device)))
    m = neuzip.MX4Manager()
    model = torch.nn.Sequential(torch.nn.Linear(64, 4, bias=False, device="meta"))
    m.load_converted(model, {"0._extra_state": blob_of(), "0._p": torch.zeros(0)}, device="cpu")
    assert went == [("0", "cpu")]
    m.import_entry(blob_of(), "0")
    assert went[1] == ("0", None)


@pytest.mark.parametrize("dtype", ("bfloat16", "float16"))
def test_a_loaded_layer_has_the_type_that_was_written(monkeypatch, dtype):
    from neuzip_b200.mx4 import MX4Backend
    monkeypatch.setattr(MX4Backend, "import_entry", lambda self, name, blob, device=None: None)
    lin = neuzip.nn.Linear.from_compressed(neuzip.MX4Manager(), blob_of(dtype=dtype), device="cpu")
    assert lin.weight.dtype == getattr(torch, dtype)


def test_the_status_word_is_not_made_inside_a_capture(monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: True)
    be = neuzip.MX4Manager()._be
    with pytest.raises(RuntimeError, match="before the capture"):
        be._status_of(0)
    be._status[0] = word = torch.zeros(1, dtype=torch.int32)
    assert be._status_of(0) is word


def test_way_of_running_of_calls_with_nothing_to_run():
    from neuzip_b200 import _lib
    L = _lib.load()
    for sizes in ((1, 0, 64, 4), (1, 64, 0, 4), (1, 64, 64, 0), (0, 64, 64, 4)):
        assert L.nz_mx4_linear_way(*sizes, 0) == -1
    assert L.nz_mx4_linear_way(1, 64, 64, 1, 0) == _lib.NZ_MX4_FEW_ROWS


def test_bytes_of_tensors_that_fill_no_tile():
    # what the module's text says: bits an element
    for shape, bits in (((128, 256), 4.25), (((128, 32)), 6.0), ((4096,), 544.0), ((8, 16, 4096), 34.0)):
        m = manager_with(shape)
        assert m.size("w") * 8 / torch.Size(shape).numel() == bits


@pytest.mark.parametrize("dtype", ("nonsense", "load", "float32"))
def test_a_layer_of_an_unknown_type_is_refused_by_the_import(dtype):
    with pytest.raises(ValueError, match="type"):
        neuzip.nn.Linear.from_compressed(neuzip.MX4Manager(), blob_of(dtype="bfloat16") | {"dtype": dtype}, device="cpu")


def test_way_of_running_of_sizes_that_the_product_refuses():
    from neuzip_b200 import _lib
    way = _lib.load().nz_mx4_linear_way
    for sizes in ((1, 1 << 31, 64, 4, 0), (1, 64, 1 << 31, 4, 0), (1, 64, 64, 1 << 31, 0), (2, 64, 64, 4, 0),
                  (8193, 64, 64, 4, 1), (1 << 40, 1 << 40, 1 << 40, 1 << 40, 1), (1, 64, 64, (1 << 64) - 1, 0)):
        assert way(*sizes) == -1, sizes
    assert way(8192, 64, 64, 4, 1) == _lib.NZ_MX4_FEW_ROWS


def test_captured_bytes_are_not_released_inside_a_capture(monkeypatch):
    m = manager_with((128, 32))
    entry = m._be.entry("w")
    m._be._captured[entry.packed.data_ptr()] = entry.packed
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: True)
    with pytest.raises(RuntimeError, match="inside the capture"):
        m.release_captured()
    assert len(m._be._captured) == 1


def test_threads_that_come_first_together_share_one_status_word(monkeypatch):
    be = neuzip.MX4Manager()._be
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: False)
    monkeypatch.setattr(be, "_lib", type("L", (), {"nz_device_check": lambda self: 0})())
    order = []
    monkeypatch.setattr(torch.cuda, "current_stream",
                        lambda device: type("S", (), {"synchronize": lambda self: order.append("cleared")})())
    zeros = torch.zeros

    def made(*shape, dtype, device):
        monkeypatch.setattr(torch, "zeros", lambda *s, dtype, device: zeros(*s, dtype=dtype))
        other.append(be._status_of(0))                       # the other thread, meanwhile
        assert order == ["cleared"]
        return zeros(*shape, dtype=dtype)
    other = []
    monkeypatch.setattr(torch, "zeros", made)
    assert be._status_of(0) is other[0] is be._status[0] and order == ["cleared"] * 2
