"""4-bit storage and its products against the definition in 64 bits (tests/mx4ref.py)."""
import pytest
import torch

import neuzip
from neuzip_b200 import _lib
from tests import mx4ref

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def rand(seed, *shape, dtype=BF16, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


# ------------------------------------------------------------------ storage
@pytest.mark.parametrize("dtype", (BF16, FP16))
@pytest.mark.parametrize("shape", [(1, 1), (1, 31), (3, 32), (5, 33), (128, 256), (129, 257), (130, 100),
                                   (3, 5, 65), (2, 128, 64), (7,), (2, 3, 4, 40), (0, 64), (300, 1000)])
def test_round_trip_is_the_definition(shape, dtype):
    m = neuzip.MX4Manager()
    w = rand(1, *shape, dtype=dtype)
    h = m.write(w.cuda())
    got = m.read(h)
    assert got.shape == w.shape and got.dtype == dtype and not got.requires_grad
    if w.numel():
        assert torch.equal(got.cpu().double(), mx4ref.quantize(w))       # the numbers of the format fit bf16
    m.check()


@pytest.mark.parametrize("dtype", (BF16, FP16))
def test_every_pattern_of_16_bits(dtype):
    # every value as the largest of a block, next to smaller ones: subnormals, ties, infinities, NaN
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
    top = bits.view(dtype).reshape(-1, 1)
    parts = torch.tensor([[1, .5, .25, .125, .0625, .3125, .1875, -.4375, -.625, 0, -0.0, 1 / 3]], dtype=dtype)
    w = (top.float() * parts.float()).to(dtype)
    m = neuzip.MX4Manager()
    got = m.read(m.write(w.cuda())).cpu()
    want = mx4ref.quantize(w)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    assert torch.equal(got.double()[~nan], want.to(dtype).double()[~nan])


def test_views_and_unaligned_tensors():
    m = neuzip.MX4Manager()
    base = rand(2, 70, 200).cuda()
    for w in (base[3:, 1:129], base.t(), base[::2], base.view(-1)[1:13901].view(139, 100)):
        assert torch.equal(m.read(m.write(w)).cpu().double(), mx4ref.quantize(w))


def test_size_replace_and_erase():
    m = neuzip.MX4Manager()
    h = m.write(rand(3, 256, 512).cuda())
    assert m.size(h) == 256 * 512 * 17 // 32 and m.total_size() == m.size(h)
    w = rand(4, 20, 40, dtype=FP16)
    assert m.write(w.cuda(), h) == h
    assert torch.equal(m.read(h).cpu().double(), mx4ref.quantize(w))
    assert m.size("unknown") == 0
    m._be.erase(h)
    with pytest.raises(RuntimeError, match="Data not found"):
        m.read(h)


@pytest.mark.parametrize("shape", [(50, 64), (50, 33), (20, 3, 40)])
def test_read_rows(shape):
    m = neuzip.MX4Manager()
    w = rand(5, *shape)
    h = m.write(w.cuda())
    want = mx4ref.quantize(w)
    for ids in (torch.tensor([[0, 3, 3], [19, 1, 0]]), torch.tensor([], dtype=torch.int64), torch.tensor(7),
                torch.arange(19, -1, -1, dtype=torch.int32)):
        got = m.read_rows(h, ids.cuda())
        assert got.shape == ids.shape + w.shape[1:]
        assert torch.equal(got.cpu().double(), want[ids.long()])
    m.check()


def test_read_rows_outside_the_table():
    m = neuzip.MX4Manager()
    w = rand(6, 50, 64)
    h = m.write(w.cuda())
    got = m.read_rows(h, torch.tensor([50, 2, -1]).cuda()).cpu()
    assert not got[0].any() and not got[2].any() and torch.equal(got[1].double(), mx4ref.quantize(w)[2])
    with pytest.raises(_lib.NeuzipError, match="out of range"):
        m.check()
    with pytest.raises(TypeError):
        m.read_rows(h, torch.tensor([1.0]).cuda())


def test_export_and_import():
    m, other = neuzip.MX4Manager(), neuzip.MX4Manager()
    w = rand(7, 3, 33, 70, dtype=FP16)
    blob = m.export_entry(m.write(w.cuda()))
    h = other.import_entry(blob)
    assert other.read(h).dtype == FP16 and torch.equal(other.read(h).cpu().double(), mx4ref.quantize(w))


# ------------------------------------------------------------------ product
def check_linear(x, w, bias=None, xd=None):
    m = neuzip.MX4Manager()
    h = m.write(w.cuda())
    y = m.linear(h, x.cuda() if xd is None else xd, None if bias is None else bias.cuda())
    assert y.dtype == x.dtype and y.shape == x.shape[:-1] + (w.shape[0],)
    want, bound = mx4ref.product(x.reshape(-1, x.shape[-1]), w, bias)
    mx4ref.check(y.reshape(-1, w.shape[0]), want, bound)
    return m, h, y


ROWS = (1, 2, 15, 16, 17, 33, 100, 129, 241, 500)


@pytest.mark.parametrize("rows", ROWS)
def test_linear_rows(rows):
    check_linear(rand(10, rows, 512), rand(11, 384, 512, scale=0.02))


@pytest.mark.parametrize("dtype", (BF16, FP16))
@pytest.mark.parametrize("out,inner", [(1, 1), (7, 31), (128, 32), (129, 64), (64, 65), (300, 100), (127, 256),
                                       (257, 257), (96, 1000), (1001, 333), (64, 2080), (130, 4160)])
@pytest.mark.parametrize("rows", (1, 5, 40, 260))
def test_linear_sizes(rows, out, inner, dtype):
    x, w = rand(12, rows, inner, dtype=dtype), rand(13, out, inner, dtype=dtype, scale=0.1)
    check_linear(x, w, rand(14, out, dtype=dtype) if (rows + out) % 2 else None)


def test_linear_larger():
    check_linear(rand(15, 700, 2048), rand(16, 1536, 2048, scale=0.02), rand(17, 1536))


@pytest.mark.parametrize("shape", [(64,), (1, 64), (2, 3, 64), (2, 0, 64), (1, 1, 1, 64)])
def test_linear_leading_dimensions(shape):
    check_linear(rand(18, *shape), rand(19, 48, 64))


def test_linear_strided_inputs():
    w = rand(20, 200, 96)
    big = rand(21, 40, 300)
    d = big.cuda()
    for lo in (8, 3, 1, 16):
        check_linear(big[:, lo:lo + 96].contiguous(), w, xd=d[:, lo:lo + 96])
        check_linear(big[::2, lo:lo + 96].contiguous(), w, xd=d[::2, lo:lo + 96])
    check_linear(big[4:5, 3:99].expand(9, 96).contiguous(), w, xd=d[4:5, 3:99].expand(9, 96))
    check_linear(big[:, :192:2].contiguous(), w, xd=d[:, :192:2])
    wide = rand(22, 96, 30)
    check_linear(wide.t().contiguous(), w, xd=wide.cuda().t())


def test_linear_mixed_types():
    # the weights' type does not matter: the result has the inputs' type
    check_linear(rand(23, 9, 128), rand(24, 40, 128, dtype=FP16))
    check_linear(rand(25, 9, 128, dtype=FP16), rand(26, 40, 128))


def test_linear_scales_far_apart():
    # block scales over a wide range of powers of two, in both operands
    e = torch.arange(32).repeat_interleave(32)
    x = rand(27, 20, 1024) * torch.exp2((e % 7 - 3).float() * 9).to(BF16)
    w = rand(28, 150, 1024) * torch.exp2((e % 5 - 2).float() * 11).to(BF16)
    check_linear(x, w)


def test_linear_zero_and_nonfinite_rows():
    x, w = rand(29, 40, 320), rand(30, 200, 320)
    x[3] = 0
    x[5, 7] = float("inf")
    x[6, 319] = float("nan")
    w[9, 100] = float("-inf")
    w[10] = 0
    _, _, y = check_linear(x, w)
    y = y.cpu()
    assert torch.isnan(y[5]).all() and torch.isnan(y[6]).all() and torch.isnan(y[:, 9]).all()
    assert not torch.isnan(y[[4, 7]][:, [8, 10, 11]]).any()


def test_linear_gives_the_same_bits_again():
    m = neuzip.MX4Manager()
    for rows, out, inner in ((1, 4096, 4096), (16, 1408, 2048), (300, 1000, 2048)):
        h = m.write(rand(31, out, inner).cuda())
        x = rand(32, rows, inner).cuda()
        first = m.linear(h, x)
        for _ in range(5):
            assert torch.equal(m.linear(h, x), first)


@pytest.mark.parametrize("rows,out,inner", [
    (1, 1200, 4096), (2, 1000, 4000), (3, 300, 8192), (1, 3500, 8192), (7, 513, 5000), (16, 2048, 2048),
    (24, 140, 16400), (64, 2000, 1024), (200, 4100, 260), (1500, 1030, 288), (1201, 2049, 96), (2600, 520, 1056)])
def test_linear_every_way_of_running(rows, out, inner):
    """Few rows, one launch, shared tiles, whole tiles, pairs: the sizes at which each is taken."""
    check_linear(rand(100, rows, inner), rand(101, out, inner, scale=0.05), rand(102, out) if rows % 2 else None)


@pytest.mark.parametrize("rows", (1, 40, 700))
@pytest.mark.parametrize("a,b", [(1e30, 1e-30), (3e38, 1e-37), (1e-30, 1e30), (1e-39, 1e36), (1e-37, 1e-2),
                                 (1e36, 1e-39)])
def test_linear_at_the_ends_of_the_range(rows, a, b):
    # scales whose product is an ordinary number, and sums that stay in range
    x = (rand(103, rows, 256, dtype=torch.float32).clamp(-3, 3) / 3 * a).to(BF16)
    w = (rand(104, 300, 256, dtype=torch.float32).clamp(-3, 3) / 3 * b).to(BF16)
    check_linear(x, w)


@pytest.mark.parametrize("rows", (1, 2, 40, 700))
@pytest.mark.parametrize("power", (125, 126, 127, 128, 140, -120, -126, -130, -133, -140))
def test_linear_results_whose_scales_leave_the_range(rows, power):
    # the largest numbers of the blocks meet zeros; what is left, 1/2 times 1/2 of the scales, is 2^power
    a = power // 2
    w, x = torch.zeros(3, 64), torch.zeros(rows, 64)
    w[:, 0], w[:, 2] = 2.0 ** (a + 3), 2.0 ** a
    x[:, 1], x[:, 2] = 2.0 ** (power - a + 3), -2.0 ** (power - a)
    m = neuzip.MX4Manager()
    y = m.linear(m.write(w.to(BF16).cuda()), x.to(BF16).cuda()).cpu()
    want = torch.full((rows, 3), -2.0 ** power, dtype=torch.float64).to(BF16)       # infinite, and 0, beyond bf16
    assert torch.equal(y, want)


def test_linear_outputs_and_inputs_beyond_32_bits():
    m = neuzip.MX4Manager()
    w = rand(105, 32768, 64)
    h = m.write(w.cuda())
    x = rand(106, 64, 64).cuda().repeat(1100, 1)              # y: 70400 x 32768 elements, over 2^31
    y = m.linear(h, x)
    want, bound = mx4ref.product(x[:4].cpu(), w)
    for r in (0, 64 * 511, 64 * 1023, 64 * 1099):
        mx4ref.check(y[r:r + 4], want, bound)
    del y, x
    w = rand(107, 40, 65536)
    h = m.write(w.cuda())
    x = rand(108, 2, 65536).cuda().repeat(16500, 1)           # x: over 2^32 bytes
    y = m.linear(h, x)
    want, bound = mx4ref.product(x[:2].cpu(), w)
    for r in (0, 16382, 32766, 32998):
        mx4ref.check(y[r:r + 2], want, bound)


def test_linear_bias_with_gaps():
    w, x, b = rand(109, 130, 96), rand(110, 20, 96), rand(111, 260)
    m = neuzip.MX4Manager()
    y = m.linear(m.write(w.cuda()), x.cuda(), b.cuda()[::2])
    want, bound = mx4ref.product(x, w, b[::2])
    mx4ref.check(y, want, bound)


# ------------------------------------------------------------------ grouped
def check_grouped(x, w, ids, bias=None):
    m = neuzip.MX4Manager()
    h = m.write(w.cuda())
    y = m.grouped_linear(h, x.cuda(), ids.cuda(), None if bias is None else bias.cuda())
    assert y.dtype == x.dtype and y.shape == ids.shape + (w.shape[1],)
    y = y.cpu()
    rows = x if x.dim() == ids.dim() + 1 else x.unsqueeze(-2).expand(ids.shape + x.shape[-1:])
    for e in range(w.shape[0]):
        at = ids == e
        if at.any():
            want, bound = mx4ref.product(rows[at], w[e], None if bias is None else bias[e])
            mx4ref.check(y[at], want, bound)
    assert not y[ids < 0].any()
    m.check()


def routes(seed, tokens, k, experts):
    g = torch.Generator().manual_seed(seed)
    return torch.rand(tokens, experts, generator=g).topk(k, dim=-1).indices


@pytest.mark.parametrize("shared", (True, False))
@pytest.mark.parametrize("tokens,k,experts,out,inner", [
    (1, 1, 1, 40, 64), (1, 2, 8, 128, 256), (3, 2, 4, 129, 100), (16, 8, 64, 96, 320), (50, 3, 13, 101, 333),
    (200, 2, 2, 256, 512), (333, 4, 7, 70, 1000), (64, 1, 128, 64, 64), (2000, 2, 5, 130, 96),
    (5, 6, 300, 33, 40)])
def test_grouped_sizes(tokens, k, experts, out, inner, shared):
    x = rand(40, *((tokens, inner) if shared else (tokens, k, inner)))
    check_grouped(x, rand(41, experts, out, inner, scale=0.1), routes(42, tokens, k, experts),
                  rand(43, experts, out) if out % 2 else None)


@pytest.mark.parametrize("tokens,k,experts", [(512, 2, 256), (1024, 1, 3), (1025, 1, 3), (205, 5, 257), (129, 8, 256),
                                              (64, 1, 70), (65, 1, 70), (300, 9, 9), (1, 8, 8), (3000, 1, 2)])
def test_grouped_limits(tokens, k, experts):
    """Around the numbers of rows and matrices at which another way of grouping is taken."""
    check_grouped(rand(112, tokens, 72), rand(113, experts, 24, 72), routes(114, tokens, k, experts))


@pytest.mark.parametrize("tokens,k,experts,out,inner", [(1, 2, 4, 600, 8192), (2, 1, 2, 2100, 4096), (30, 4, 16, 400, 1024),
                                                        (600, 2, 4, 520, 544), (900, 3, 3, 257, 1000)])
def test_grouped_every_way_of_running(tokens, k, experts, out, inner):
    check_grouped(rand(115, tokens, inner), rand(116, experts, out, inner, scale=0.05), routes(117, tokens, k, experts),
                  rand(118, experts, out))


def test_grouped_many_rows_without_an_expert():
    ids = torch.randint(-1, 5, (1400, 3), generator=torch.Generator().manual_seed(119))
    check_grouped(rand(120, 1400, 100), rand(121, 5, 131, 100), ids)
    ids[:] = -1
    check_grouped(rand(122, 1400, 100), rand(121, 5, 131, 100), ids)


def test_grouped_numbers_outside_a_large_stack():
    m = neuzip.MX4Manager()
    w = rand(123, 3, 20, 64)
    h = m.write(w.cuda())
    ids = torch.randint(0, 3, (2000,), generator=torch.Generator().manual_seed(124))
    ids[7], ids[1999] = 3, -5
    x = rand(125, 2000, 64)
    y = m.grouped_linear(h, x.cuda(), ids.cuda()).cpu()
    assert not y[7].any() and not y[1999].any()
    for e in range(3):
        mx4ref.check(y[ids == e], *mx4ref.product(x[ids == e], w[e]))
    with pytest.raises(_lib.NeuzipError, match="out of range"):
        m.check()
    with pytest.raises(ValueError, match="at most"):
        big = m.write(torch.zeros(8193, 1, 32, dtype=BF16, device="cuda"))
        m.grouped_linear(big, x[:, :32].cuda(), ids.cuda())


def test_grouped_strided_inputs():
    m = neuzip.MX4Manager()
    w = rand(126, 5, 40, 96)
    h = m.write(w.cuda())
    wide = rand(127, 50, 300)
    ids = routes(128, 50, 2, 5)
    for lo in (0, 1, 8, 16):
        y = m.grouped_linear(h, wide.cuda()[:, lo:lo + 96], ids.cuda().t().contiguous().t()).cpu()
        for j in range(2):
            for e in range(5):
                at = ids[:, j] == e
                if at.any():
                    mx4ref.check(y[at, j], *mx4ref.product(wide[at, lo:lo + 96], w[e]))


def test_grouped_fp16_and_int32():
    check_grouped(rand(44, 30, 100, dtype=FP16), rand(45, 6, 50, 100, dtype=FP16),
                  routes(46, 30, 2, 6).to(torch.int32), rand(47, 6, 50, dtype=FP16))


def test_grouped_rows_without_an_expert():
    ids = routes(48, 70, 2, 5)
    ids[::3] = -1
    ids[4, 1] = -1
    check_grouped(rand(49, 70, 128), rand(50, 5, 200, 128), ids, rand(51, 5, 200))
    check_grouped(rand(52, 70, 2, 128), rand(50, 5, 200, 128), ids)
    check_grouped(rand(53, 9, 128), rand(50, 5, 200, 128), torch.full((9, 2), -1))


def test_grouped_one_expert_takes_all():
    check_grouped(rand(54, 300, 64), rand(55, 9, 130, 64), torch.full((300, 1), 8))
    check_grouped(rand(56, 20, 64), rand(55, 9, 130, 64), torch.full((20, 3), 4))      # the same expert twice


def test_grouped_other_ranks():
    w = rand(57, 4, 30, 64)
    check_grouped(rand(58, 64), w, torch.tensor(3))
    check_grouped(rand(59, 64), w, torch.tensor([3, 0]))
    check_grouped(rand(60, 2, 3, 64), w, torch.tensor([[[0, 1], [2, 3], [-1, 0]], [[3, 3], [1, 2], [0, 2]]]))
    check_grouped(rand(61, 7, 64), w, torch.tensor([0, 1, 2, 3, 0, 0, -1]))


def test_grouped_numbers_outside_the_stack():
    m = neuzip.MX4Manager()
    w = rand(62, 4, 30, 64)
    h = m.write(w.cuda())
    x = rand(63, 5, 64)
    y = m.grouped_linear(h, x.cuda(), torch.tensor([0, 4, -2, 2 ** 40, 3]).cuda()).cpu()
    assert not y[1:4].any()
    for r, e in ((0, 0), (4, 3)):
        mx4ref.check(y[r:r + 1], *mx4ref.product(x[r:r + 1], w[e]))
    with pytest.raises(_lib.NeuzipError, match="out of range"):
        m.check()


def test_grouped_gives_the_same_bits_again():
    m = neuzip.MX4Manager()
    h = m.write(rand(64, 16, 300, 512).cuda())
    for tokens in (2, 500):
        x, ids = rand(65, tokens, 512).cuda(), routes(66, tokens, 4, 16).cuda()
        first = m.grouped_linear(h, x, ids)
        for _ in range(5):
            assert torch.equal(m.grouped_linear(h, x, ids), first)


# ------------------------------------------------------------------ as a program uses them
def test_layer_with_experts():
    """Embedding, dense projection, experts up and down, gated sum: one run of all of them."""
    m = neuzip.MX4Manager()
    g = torch.Generator().manual_seed(70)
    table, dense = torch.nn.Embedding(100, 128, dtype=BF16), torch.nn.Linear(128, 192, dtype=BF16)
    matrix, vector = dense.weight.detach().clone(), dense.bias.detach().clone()   # convert drops them
    up, down = rand(71, 6, 160, 192, scale=0.1), rand(72, 6, 192, 160, scale=0.1)
    tokens = torch.randint(0, 100, (2, 9), generator=g)
    emb = neuzip.nn.Embedding(m, table.cuda())
    model = torch.nn.Sequential(dense).cuda()
    m.convert(model)
    assert isinstance(model[0], neuzip.nn.Linear)
    e_up, e_down = neuzip.nn.Experts(m, up.cuda()), neuzip.nn.Experts(m, down.cuda())
    ids = routes(73, 18, 2, 6).view(2, 9, 2)
    gate = torch.rand(2, 9, 2, 1, generator=g).to(BF16)
    with torch.no_grad():
        h0 = emb(tokens.cuda())
        assert torch.equal(h0.cpu().double(), mx4ref.quantize(table.weight)[tokens])
        h1 = model(h0)
        want, bound = mx4ref.product(h0.cpu().view(-1, 128), matrix, vector)
        mx4ref.check(h1.view(-1, 192), want, bound)
        u = e_up(h1, ids.cuda())
        h2 = torch.relu(u)
        h3 = e_down(h2, ids.cuda())
        y = (h3 * gate.cuda()).sum(-2)
    assert y.shape == (2, 9, 192)
    for (a, b, k), e in zip([(a, b, k) for a in range(2) for b in range(9) for k in range(2)],
                            ids.reshape(-1).tolist()):
        mx4ref.check(u[a, b, k:k + 1], *mx4ref.product(h1[a, b:b + 1].cpu(), up[e]))
        mx4ref.check(h3[a, b, k:k + 1], *mx4ref.product(h2[a, b, k:k + 1].cpu(), down[e]))
    m.check()


def test_checkpoint_of_a_converted_model():
    m = neuzip.MX4Manager()
    model = torch.nn.Sequential(torch.nn.Linear(64, 40, dtype=BF16)).cuda()
    dense = model[0].weight.detach().clone()
    m.convert(model)
    experts = neuzip.nn.Experts(m, rand(74, 3, 20, 40).cuda(), rand(75, 3, 20).cuda())
    state, more = model.state_dict(), experts.state_dict()
    other = neuzip.MX4Manager()
    loaded = other.load_converted(torch.nn.Sequential(torch.nn.Linear(64, 40, dtype=BF16, device="meta")), state,
                                  device="cuda")
    x = rand(76, 5, 64).cuda()
    fresh = neuzip.nn.Experts(other, torch.zeros(3, 20, 40, dtype=BF16, device="cuda"),
                              torch.zeros(3, 20, dtype=BF16, device="cuda"))
    fresh.load_state_dict(more)
    with torch.no_grad():
        assert torch.equal(loaded(x), model(x))
        assert torch.equal(loaded[0]._p().cpu().double(), mx4ref.quantize(dense))
        ids = torch.tensor([0, 1, 2, 2, 0]).cuda()
        assert torch.equal(fresh(model(x), ids), experts(model(x), ids))


def test_linear_under_autograd():
    """The framework's autograd function: gradients of the product with the stored weights, the
    inputs' rounding taken as the identity."""
    m = neuzip.MX4Manager()
    lin = torch.nn.Linear(96, 40, dtype=BF16).cuda()
    wq = mx4ref.quantize(lin.weight)
    model = m.convert(torch.nn.Sequential(lin))
    x = rand(77, 8, 96).cuda().requires_grad_()
    g = rand(78, 8, 40)
    y = model(x)
    y.backward(g.cuda())
    dx, dw = g.double() @ wq, g.double().t() @ x.detach().cpu().double()
    s = g.double().abs() @ wq.abs()
    assert ((x.grad.cpu().double() - dx).abs() <= 2.0 ** -8 * dx.abs() + 40 * 2.0 ** -23 * s).all()
    s = g.double().abs().t() @ x.detach().cpu().double().abs()
    got = model[0]._p._gradient.cpu().double()
    assert ((got - dw).abs() <= 2.0 ** -8 * dw.abs() + 8 * 2.0 ** -23 * s).all()


def test_linear_gradient_against_differences():
    """Where inputs are numbers of the format their rounding is the identity: between two such points
    the layer is linear, and its gradient is the slope."""
    m = neuzip.MX4Manager()
    model = m.convert(torch.nn.Sequential(torch.nn.Linear(64, 24, dtype=BF16, bias=False).cuda()))
    g = torch.Generator().manual_seed(79)
    points = []
    for _ in range(2):
        p = mx4ref.GRID[torch.randint(0, 8, (5, 64), generator=g)] * torch.randint(0, 2, (5, 64), generator=g).mul(2).sub(1)
        p[:, ::32] = 6                                        # every block has the scale 1
        points.append(p.to(BF16).cuda())
    up = torch.randint(-2, 3, (5, 24), generator=g).to(BF16).cuda()
    x = points[0].clone().requires_grad_()
    y0 = model(x)
    y0.backward(up)
    with torch.no_grad():
        y1 = model(points[1])
    step = (points[1] - points[0]).double()
    slope = (x.grad.double() * step).sum()
    rise = (up.double() * (y1.detach().double() - y0.detach().double())).sum()
    # both sides are sums of values rounded to bf16, each off by half a step at most
    room = 2.0 ** -8 * ((x.grad.double() * step).abs().sum()
                        + (up.double().abs() * (y1.detach().double().abs() + y0.detach().double().abs())).sum())
    assert (slope - rise).abs() <= room


def test_graph_replay_follows_its_inputs():
    m = neuzip.MX4Manager()
    w, stack = rand(80, 500, 512), rand(81, 6, 130, 512)
    h, hs = m.write(w.cuda()), m.write(stack.cuda())
    x, ids = rand(82, 20, 512).cuda(), routes(83, 20, 2, 6).cuda()
    m.linear(h, x), m.grouped_linear(hs, x, ids)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                       # two graphs, each with a workspace of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            a, b = m.linear(h, x), m.grouped_linear(hs, x, ids)
        graphs.append((graph, a, b))
    for seed in (84, 85):
        x.copy_(rand(seed, 20, 512))
        ids.copy_(routes(seed + 10, 20, 2, 6))
        for graph, _, _ in graphs:
            graph.replay()
        want = m.linear(h, x), m.grouped_linear(hs, x, ids)
        for _, a, b in graphs:
            assert torch.equal(a, want[0]) and torch.equal(b, want[1])


def test_a_graph_keeps_the_bytes_it_reads():
    m = neuzip.MX4Manager()
    w = rand(130, 300, 512)
    h = m.write(w.cuda())
    x = rand(131, 20, 512).cuda()
    want = m.linear(h, x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = m.linear(h, x)
    for seed in range(4):                    # the handle is written again, and what was freed is reused
        m.write(rand(132 + seed, 300, 512).cuda(), h)
        torch.full((300 * 512,), 255, dtype=torch.uint8, device="cuda")
    graph.replay()
    assert torch.equal(y, want)


def test_threads_share_a_manager():
    import threading
    m = neuzip.MX4Manager()
    ws = [rand(140 + i, 200 + i, 256) for i in range(4)]
    hs = [m.write(w.cuda()) for w in ws]
    x = rand(150, 33, 256).cuda()
    want = [m.linear(h, x) for h in hs]
    bad = []

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                if not torch.equal(m.linear(hs[k], x), want[k]):
                    bad.append(k)
            torch.cuda.current_stream().synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_calls_on_two_streams():
    m = neuzip.MX4Manager()
    hs = m.write(rand(86, 8, 256, 1024).cuda())
    xs = [rand(87 + i, 300, 1024).cuda() for i in range(2)]
    ids = [routes(90 + i, 300, 2, 8).cuda() for i in range(2)]
    want = [m.grouped_linear(hs, x, i) for x, i in zip(xs, ids)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(m.grouped_linear(hs, xs[k], ids[k]))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(g, want[k]) for g in got[k])


def test_rows_do_not_depend_on_their_neighbours():
    m = neuzip.MX4Manager()
    h = m.write(rand(95, 300, 600).cuda())
    x = rand(96, 50, 600).cuda()
    alone = torch.cat([m.linear(h, x[i:i + 1]) for i in range(50)])
    want, bound = mx4ref.product(x.cpu(), m.read(h).cpu())
    mx4ref.check(alone, want, bound)
    mx4ref.check(m.linear(h, x), want, bound)
