"""Layers on 4-bit storage as training and autocast use them (definition in 64 bits: tests/mx4ref.py)."""
import pytest
import torch

import neuzip
from tests import mx4ref

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def rand(seed, *shape, dtype=BF16, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def layer(out, inner, dtype=BF16, seed=300):
    """(layer on 4-bit storage, its matrix and vector before conversion)"""
    lin = torch.nn.Linear(inner, out, dtype=dtype)
    with torch.no_grad():
        lin.weight.copy_(rand(seed, out, inner, dtype=dtype, scale=0.1))
        lin.bias.copy_(rand(seed + 1, out, dtype=dtype))
    w, b = lin.weight.detach().clone(), lin.bias.detach().clone()
    return neuzip.MX4Manager().convert(torch.nn.Sequential(lin.cuda()))[0], w, b


@pytest.mark.parametrize("rows", ((1,), (3, 7), (0,)))
def test_a_bias_trains_over_a_frozen_matrix(rows):
    lin, w, b = layer(40, 96)
    lin._p.requires_grad_(False)
    x, g = rand(302, *rows, 96), rand(303, *rows, 40)
    y = lin(x.cuda())
    mx4ref.check(y.view(-1, 40), *mx4ref.product(x.view(-1, 96), w, b))
    y.backward(g.cuda())
    # a sum of n terms in fp32 and one rounding to bf16, half a step
    terms = g.double().view(-1, 40)
    want = terms.sum(0)
    room = 2.0 ** -8 * want.abs() + max(1, len(terms)) * 2.0 ** -23 * terms.abs().sum(0) * (1 + 2.0 ** -8)
    assert ((lin.bias.grad.cpu().double() - want).abs() <= room).all()
    assert lin._p._gradient is None and lin._p.grad is None
    # linear in the bias: between two points of it the results rise by the slope, up to both results' bounds
    with torch.no_grad():
        lin.bias += 1
        again = lin(x.cuda()).cpu().double().view(-1, 40)
    later = lin.bias.detach().cpu()
    first, second = mx4ref.product(x.view(-1, 96), w, b)[1], mx4ref.product(x.view(-1, 96), w, later)[1]
    rise = (terms * (again - y.detach().cpu().double().view(-1, 40))).sum()
    assert (rise - (want * (later.double() - b.double())).sum()).abs() <= (terms.abs() * (first + second)).sum()


def test_a_result_with_a_trained_bias_may_be_changed_in_place():
    lin, _, _ = layer(40, 96)
    lin._p.requires_grad_(False)
    y = lin(rand(304, 5, 96).cuda())
    y.mul_(2)
    y.sum().backward()
    assert torch.equal(lin.bias.grad.cpu(), torch.full((40,), 10, dtype=BF16))


@pytest.mark.parametrize("to", (BF16, FP16))
@pytest.mark.parametrize("needs", ("nothing", "inputs", "bias"))
def test_layers_under_autocast(to, needs):
    """fp32 inputs and an fp32 bias over a bf16 matrix, as functional.linear takes them under autocast."""
    lin, w, _ = layer(40, 96)
    lin._p.requires_grad_(needs == "inputs")
    b = rand(310, 40, dtype=torch.float32)
    lin.bias = torch.nn.Parameter(b.cuda(), requires_grad=needs != "nothing")
    x = rand(311, 9, 96, dtype=torch.float32)
    xd = x.cuda().requires_grad_(needs == "inputs")
    with torch.autocast("cuda", dtype=to):
        y = lin(xd)
    assert y.dtype == to
    mx4ref.check(y, *mx4ref.product(x.to(to), w, b.to(to)))
    if needs == "bias":
        y.sum().backward()
        assert torch.equal(lin.bias.grad.cpu(), torch.full((40,), 9.0))


@pytest.mark.parametrize("to", (BF16, FP16))
def test_experts_under_autocast(to):
    w, b = rand(312, 3, 40, 96, scale=0.1), rand(313, 3, 40, dtype=torch.float32)
    experts = neuzip.nn.Experts(neuzip.MX4Manager(), w.cuda(), b.cuda())
    x, ids = rand(314, 3, 96, dtype=torch.float32), torch.arange(3)
    with torch.autocast("cuda", dtype=to):
        y = experts(x.cuda(), ids.cuda())
    assert y.dtype == to
    for e in range(3):
        mx4ref.check(y[e:e + 1], *mx4ref.product(x[e:e + 1].to(to), w[e], b[e].to(to)))


@pytest.mark.parametrize("wide", (True, False))
@pytest.mark.parametrize("x_type,w_type", [(FP16, BF16), (BF16, FP16), (BF16, BF16), (FP16, FP16)])
def test_gradients_of_mixed_types(x_type, w_type, wide):
    """Inputs and matrix of different 16-bit types; a bf16 matrix beyond fp16's range (`wide`) with gradients that
    bring the results back into it."""
    lin, w, _ = layer(40, 96, dtype=w_type)
    scale = 2.0 ** 20 if wide and w_type == BF16 else 1.0
    lin.manager.write((w * scale).cuda(), lin._p._handle)
    wq = mx4ref.quantize(w * scale)
    lin.bias = None
    x = rand(320, 8, 96, dtype=x_type, scale=2.0 ** -12 if scale > 1 else 1.0)
    g = rand(321, 8, 40, dtype=x_type, scale=2.0 ** -12 if scale > 1 else 1.0)
    xd = x.cuda().requires_grad_()
    y = lin(xd)
    mx4ref.check(y, *mx4ref.product(x, w * scale))
    y.backward(g.cuda())
    half = torch.finfo(x_type).eps / 2
    # sums of n products in fp32, one rounding to the type of x and its smallest numbers
    for got, a, b in ((xd.grad, g.double(), wq), (lin._p._gradient, g.double().t(), x.double())):
        want, sums = a @ b, a.shape[1] * 2.0 ** -23 * (a.abs() @ b.abs())
        room = sums + half * (want.abs() + sums) + torch.finfo(x_type).smallest_normal * half
        assert got.dtype == x_type and ((got.cpu().double() - want).abs() <= room).all()


def test_bytes_of_captured_graphs_can_be_given_back():
    m = neuzip.MX4Manager()
    h = m.write(rand(330, 1024, 1024).cuda())
    x = rand(331, 20, 1024).cuda()
    m.linear(h, x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = m.linear(h, x)
    size = m.size(h)
    assert m.captured_bytes() == 0
    m.write(rand(332, 1024, 1024).cuda(), h)
    assert m.captured_bytes() == size
    graph.replay()
    want = y.clone()
    assert not torch.equal(m.linear(h, x), want)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    graph.reset()
    m.release_captured()
    assert m.captured_bytes() == 0 and torch.cuda.memory_allocated() <= before - size
    m.check()


def test_a_checkpoint_is_loaded_onto_the_devices_of_its_layers():
    m = neuzip.MX4Manager()
    w = rand(340, 24, 64)
    h = m.write(w.cuda())
    blob = m.export_entry(h)
    here = torch.device("cuda", torch.cuda.current_device())
    for name, device in ((h, None), ("a", None), ("b", "cuda"), ("c", here), ("d", "cuda:%d" % here.index)):
        m.import_entry(blob, name, device)
        assert m._be.entry(name).device == here
        assert torch.equal(m.read(name).cpu().double(), mx4ref.quantize(w))
    if torch.cuda.device_count() > 1:
        m.import_entry(blob, "e", "cuda:1")
        m.import_entry(blob, "e")
        x = rand(341, 3, 64)
        mx4ref.check(m.linear("e", x.to("cuda:1")), *mx4ref.product(x, w))
    m.check()


def test_the_first_call_of_a_manager_is_a_captured_one():
    """A write is quantised at every replay; products and row lookups need the status word, which has to be
    there before, so that no replay clears what other calls have reported."""
    from neuzip_b200 import _lib
    w, x = rand(350, 60, 96).cuda(), rand(351, 5, 96).cuda()
    m = neuzip.MX4Manager()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h = m.write(w)
        got = m.read(h)
        with pytest.raises(RuntimeError, match="before the capture"):
            m.linear(h, x)
        with pytest.raises(RuntimeError, match="before the capture"):
            m.read_rows(h, torch.zeros(1, dtype=torch.int64, device="cuda"))
    assert not m._be._status
    graph.replay()
    assert torch.equal(got.cpu().double(), mx4ref.quantize(w))
    m.check()
    m.read_rows(h, torch.tensor([60]).cuda())
    w.neg_()
    graph.replay()
    assert torch.equal(got.cpu().double(), mx4ref.quantize(w))
    with pytest.raises(_lib.NeuzipError, match="out of range"):
        m.check()


@pytest.mark.parametrize("far", (20, -1, 2 ** 62, -2 ** 62, 2 ** 63 - 1, -2 ** 63))
def test_rows_far_outside_a_table_of_several_dimensions(far):
    from neuzip_b200 import _lib
    m = neuzip.MX4Manager()
    w = rand(360, 20, 4, 40)
    h = m.write(w.cuda())
    got = m.read_rows(h, torch.tensor([far, 19]).cuda()).cpu()
    assert not got[0].any() and torch.equal(got[1].double(), mx4ref.quantize(w)[19])
    with pytest.raises(_lib.NeuzipError, match="out of range"):
        m.check()
