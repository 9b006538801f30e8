"""Every way of running the 4-bit product, at sizes that are known to take it: the way is asked of the library and
compared, so that a change of the choice cannot leave a way untested.

Matrices are compared through what `read` gives (which other tests hold to the definition), inputs through the
definition itself; sums and bounds are those of tests/mx4ref.py, computed in 64 bits on the GPU."""
import pytest
import torch

import neuzip
from neuzip_b200 import _lib
from tests import mx4ref

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
FEW, ONE, WHOLE, SHARED, PAIRS = (_lib.NZ_MX4_FEW_ROWS, _lib.NZ_MX4_ONE_LAUNCH, _lib.NZ_MX4_WHOLE_TILES,
                                  _lib.NZ_MX4_SHARED_TILES, _lib.NZ_MX4_PAIRS)


def rand(seed, *shape, dtype=BF16, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def takes(way, matrices, out, inner, n_rows, grouped):
    """The choice depends on the number of SMs: the sizes here are chosen for 148."""
    if torch.cuda.get_device_properties(0).multi_processor_count != 148:
        pytest.skip("sizes are chosen for 148 SMs")
    assert _lib.load().nz_mx4_linear_way(matrices, out, inner, n_rows, grouped) == way


def compare(y, xq, wq, bias):
    """As mx4ref.product and mx4ref.check: the bound is derived there."""
    want, s = xq @ wq.t(), xq.abs() @ wq.abs().t()
    if bias is not None:
        want, s = want + bias.double(), s + bias.double().abs()
    sums, info = (xq.shape[-1] / 32 + 2) * 2.0 ** -23 * s, torch.finfo(y.dtype)
    bound = sums + info.eps / 2 * (want.abs() + sums) + info.smallest_normal * info.eps / 2
    assert y.shape == want.shape
    over = ((y.double() - want).abs() - bound).max().item() if y.numel() else 0.0
    assert over <= 0, f"{over} over the bound"


DENSE = [
    # rows, out, inner, way: what is particular
    (1, 1031, 4100, FEW), (2, 1025, 2049, FEW),
    (8, 700, 1000, ONE), (40, 601, 641, ONE), (600, 200, 1000, ONE),
    (16, 11008, 4096, WHOLE), (1025, 130, 4160, WHOLE), (1000, 301, 4101, WHOLE), (2600, 520, 1056, WHOLE),
    (4000, 2100, 96, WHOLE),
    (24, 4100, 8192, SHARED),           # two pieces a tile
    (16, 4096, 11008, SHARED),          # four
    (40, 301, 16390, SHARED),           # eight, rows that begin anywhere, a last step of 6 columns
    (5, 130, 16390, SHARED), (100, 2049, 8192, SHARED), (400, 520, 8192, SHARED),
    (2600, 4100, 520, PAIRS),           # an odd number of tiles: the last pair's second CTA stores nothing
    (4000, 1500, 1056, PAIRS),          # a last step of one block
    (2001, 3501, 1055, PAIRS),          # nothing a multiple of anything
    (1001, 4099, 2083, PAIRS),
    (500, 4100, 4160, PAIRS),           # 17 steps: the ring of stages goes round
    (1041, 3500, 2080, PAIRS),          # a last slot of 145 rows
    (2017, 2049, 2080, PAIRS),          # a last slot of 97 rows, a last tile of one row of W
    (1500, 8200, 520, PAIRS),
    (4001, 4100, 288, PAIRS),           # a last slot of 161 rows of 240
]


@pytest.mark.parametrize("rows,out,inner,way", DENSE)
def test_dense(rows, out, inner, way):
    takes(way, 1, out, inner, rows, 0)
    dtype = FP16 if out % 2 else BF16
    m = neuzip.MX4Manager()
    h = m.write(rand(1, out, inner, dtype=dtype, scale=0.05))
    x = rand(2, rows, inner, dtype=dtype)
    bias = rand(3, out, dtype=dtype) if rows % 2 or out % 4 == 0 else None
    y = m.linear(h, x, bias)
    compare(y, mx4ref.quantize(x).cuda(), m.read(h).double(), bias)
    for _ in range(3):
        assert torch.equal(m.linear(h, x, bias), y)
    m.check()


@pytest.mark.parametrize("rows,out,inner,way", [(40, 601, 640, ONE), (2600, 520, 1056, WHOLE), (100, 2049, 8192, SHARED),
                                                (2600, 4100, 520, PAIRS)])
def test_dense_strided_inputs(rows, out, inner, way):
    takes(way, 1, out, inner, rows, 0)
    m = neuzip.MX4Manager()
    h = m.write(rand(4, out, inner, scale=0.05))
    wide = rand(5, rows, inner + 40)
    for lo in (0, 1, 8, 16):
        x = wide[:, lo:lo + inner]
        compare(m.linear(h, x), mx4ref.quantize(x).cuda(), m.read(h).double(), None)


@pytest.mark.parametrize("rows,out,inner,way", [(2, 1025, 2049, FEW), (40, 601, 640, ONE), (2600, 520, 1056, WHOLE),
                                                (100, 2049, 8192, SHARED), (2600, 4100, 520, PAIRS)])
def test_rows_do_not_see_their_neighbours(rows, out, inner, way):
    """The same way of running, the other rows replaced by very large numbers, infinities and NaN: a row that stays
    keeps its bits."""
    takes(way, 1, out, inner, rows, 0)
    m = neuzip.MX4Manager()
    h = m.write(rand(6, out, inner, scale=0.05))
    x = rand(7, rows, inner)
    y = m.linear(h, x)
    stay = torch.zeros(rows, dtype=torch.bool, device="cuda")
    stay[::3] = True
    stay[-1] = rows > 2
    for value in (3e38, float("inf"), float("nan")):
        z = torch.where(stay[:, None], x, torch.full_like(x, value))
        got = m.linear(h, z)
        assert torch.equal(got[stay], y[stay])
        assert value == 3e38 or torch.isnan(got[~stay]).all()


@pytest.mark.parametrize("rows,out,inner,way", [(600, 200, 1000, ONE), (2600, 520, 1056, WHOLE), (100, 2049, 8192, SHARED),
                                                (2600, 4100, 520, PAIRS)])
def test_rows_that_share_an_input_without_matrix_numbers(rows, out, inner, way):
    """Straight from the library: y[r] = x[r / per_input] W^T, x without a row more than that."""
    takes(way, 1, out, inner, rows, 0)
    L, m = _lib.load(), neuzip.MX4Manager()
    h = m.write(rand(8, out, inner, scale=0.05))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    need = int(L.nz_mx4_linear_workspace_bytes(1, out, inner, rows, 0))
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    for per_input in (2, 5, rows):
        if rows % per_input:
            continue
        x = rand(9, rows // per_input, inner)
        y = torch.empty(rows, out, dtype=BF16, device="cuda")
        _lib.check(L.nz_mx4_linear(m._be.entry(h).packed.data_ptr(), 1, out, inner, _lib.NZ_DTYPE_BF16, x.data_ptr(),
                                   inner, rows, per_input, None, None, y.data_ptr(), ws.data_ptr(), need,
                                   status.data_ptr(), torch.cuda.current_stream().cuda_stream))
        want = m.linear(h, x.repeat_interleave(per_input, 0))
        assert torch.equal(y, want)
    assert status.item() == 0


# ------------------------------------------------------------------ grouped
GROUPED = [
    # matrices, out, inner, tokens, k, way
    (4, 300, 640, 4, 2, FEW),
    (4, 401, 1000, 50, 2, ONE), (10, 1031, 4161, 6, 2, ONE),
    (70, 1030, 288, 64, 2, WHOLE),      # grouped in every block
    (300, 131, 288, 64, 2, WHOLE),      # grouped by a kernel of its own: many matrices
    (8, 1001, 1000, 777, 3, WHOLE),     # many rows
    (2, 1030, 8192, 2, 2, SHARED),      # in every block
    (3, 1031, 8190, 2, 2, SHARED),
    (8, 520, 8192, 1, 8, SHARED),
    (4, 65, 8192, 350, 2, SHARED),
    (2, 301, 16390, 50, 2, SHARED),     # six pieces a tile
    (5, 64, 8192, 750, 2, SHARED),      # by a kernel of its own
    (5, 67, 8191, 750, 2, SHARED),
    (16, 4100, 288, 1300, 2, PAIRS),    # an odd number of tiles
    (5, 130, 4160, 5000, 2, PAIRS),
    (7, 1001, 1055, 2000, 3, PAIRS),    # nothing a multiple of anything
    (4, 1031, 2083, 2500, 2, PAIRS),
    (3, 2049, 1056, 2000, 2, PAIRS),    # a last step of one block, a last tile of one row
]


def check_grouped(m, h, w, x, ids, bias):
    y = m.grouped_linear(h, x, ids, bias)
    rows = (x if x.dim() == ids.dim() + 1 else x.unsqueeze(-2).expand(ids.shape + x.shape[-1:])).reshape(-1, x.shape[-1])
    xq, flat, got = mx4ref.quantize(rows).cuda(), ids.reshape(-1), y.reshape(-1, y.shape[-1])
    for e in range(w.shape[0]):
        at = flat == e
        if at.any():
            compare(got[at], xq[at], w[e].double(), None if bias is None else bias[e])
    assert not got[(flat < 0) | (flat >= w.shape[0])].any()
    return y


@pytest.mark.parametrize("shared", (True, False))
@pytest.mark.parametrize("matrices,out,inner,tokens,k,way", GROUPED)
def test_grouped(matrices, out, inner, tokens, k, way, shared):
    takes(way, matrices, out, inner, tokens * k, 1)
    dtype = FP16 if out % 2 else BF16
    m = neuzip.MX4Manager()
    h = m.write(rand(20, matrices, out, inner, dtype=dtype, scale=0.05))
    w = m.read(h)
    x = rand(21, *((tokens, inner) if shared else (tokens, k, inner)), dtype=dtype)
    bias = rand(22, matrices, out, dtype=dtype) if out % 2 or matrices % 2 else None
    g = torch.Generator(device="cuda").manual_seed(23)
    ids = torch.rand(tokens, matrices, generator=g, device="cuda").topk(k, dim=-1).indices
    y = check_grouped(m, h, w, x, ids, bias)
    for _ in range(3):
        assert torch.equal(m.grouped_linear(h, x, ids, bias), y)
    # some rows without a matrix, whole tokens and single ones; uneven numbers of rows
    gaps = torch.where(torch.rand(tokens, k, generator=g, device="cuda") < 0.3, -1, ids)
    gaps[::5] = -1
    check_grouped(m, h, w, x, gaps, bias)
    # one matrix takes all; nobody has one
    check_grouped(m, h, w, x, torch.full_like(ids, matrices - 1), bias)
    check_grouped(m, h, w, x, torch.full_like(ids, -1), bias)
    m.check()
    gaps[0, 0], gaps[-1, -1] = matrices, -2
    check_grouped(m, h, w, x, gaps, bias)
    with pytest.raises(_lib.NeuzipError, match="out of range"):
        m.check()


@pytest.mark.parametrize("matrices,out,inner,rows", [(13, 641, 16390, 15), (20, 520, 12300, 20)])
def test_shared_tiles_when_more_matrices_are_named_than_expected(matrices, out, inner, rows):
    """The plan expects that rows meet in some matrices and divides its tiles into pieces; where every matrix is
    named there are more than one tile for two CTAs, and all steps are divided evenly instead."""
    takes(SHARED, matrices, out, inner, rows, 1)
    m = neuzip.MX4Manager()
    h = m.write(rand(30, matrices, out, inner, scale=0.05))
    w, x = m.read(h), rand(31, rows, inner)
    assert 2 * matrices * -(-out // 128) > 148
    every = torch.arange(rows, device="cuda") % matrices
    y = check_grouped(m, h, w, x, every, None)
    for _ in range(20):
        assert torch.equal(m.grouped_linear(h, x, every), y)
    check_grouped(m, h, w, x, torch.where(every == 3, -1, every), None)


def test_graphs_of_every_way_replay():
    m = neuzip.MX4Manager()
    calls = []
    for rows, out, inner, way in ((1, 1031, 4100, FEW), (40, 601, 641, ONE), (2600, 520, 1056, WHOLE),
                                  (40, 301, 16390, SHARED), (2600, 4100, 520, PAIRS)):
        takes(way, 1, out, inner, rows, 0)
        h, x = m.write(rand(40, out, inner, scale=0.05)), rand(41, rows, inner)
        calls.append((x, lambda h=h, x=x: m.linear(h, x)))
    for matrices, out, inner, tokens, k, way in ((5, 64, 8192, 750, 2, SHARED), (3, 2049, 1056, 2000, 2, PAIRS)):
        h, x = m.write(rand(42, matrices, out, inner, scale=0.05)), rand(43, tokens, inner)
        ids = torch.randint(-1, matrices, (tokens, k), device="cuda")
        calls.append((x, lambda h=h, x=x, ids=ids: m.grouped_linear(h, x, ids)))
    for _, call in calls:
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [call() for _, call in calls]
    for seed in (44, 45):
        for x, _ in calls:
            x.copy_(rand(seed, *x.shape))
        graph.replay()
        for y, (_, call) in zip(got, calls):
            assert torch.equal(y, call())
    m.check()
