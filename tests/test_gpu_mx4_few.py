"""The 4-bit product for few rows where a CTA takes several items, some of them without a matrix."""
import pytest
import torch

import neuzip
from neuzip_b200 import _lib
from tests import mx4ref

pytestmark = pytest.mark.gpu


def rand(seed, *shape, dtype=torch.bfloat16, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("out,inner", [(1280, 2304), (1408, 2080)])
@pytest.mark.parametrize("missing", [{3: -1}, {4: -1}, {3: 9, 4: -1}, {0: -1, 3: -1, 4: 77, 7: -1}])
def test_rows_without_a_matrix_between_rows_of_one_input(missing, out, inner, dtype):
    """One token to eight matrices is 320 and 352 items here, up to three for a CTA, all of the same input row:
    where the middle one has no matrix, nothing but its place lies between the sums of the other two."""
    w, x, ids = rand(200, 8, out, inner, dtype=dtype, scale=0.05), rand(201, 1, inner, dtype=dtype), torch.arange(8)
    for at, number in missing.items():
        ids[at] = number
    m = neuzip.MX4Manager()
    h = m.write(w.cuda())
    xd, idd = x.cuda(), ids.view(1, 8).cuda()
    first = m.grouped_linear(h, xd, idd)
    for r in range(8):
        if r in missing:
            assert not first[0, r].any()
        else:
            mx4ref.check(first[0, r:r + 1], *mx4ref.product(x, w[r]))
    for _ in range(200):
        assert torch.equal(m.grouped_linear(h, xd, idd), first)
    if any(number > 0 for number in missing.values()):
        with pytest.raises(_lib.NeuzipError, match="out of range"):
            m.check()
    else:
        m.check()


@pytest.mark.parametrize("n_rows,per_input", [(1, 1), (2, 1), (2, 2), (4, 4), (40, 2), (40, 40), (600, 3), (2600, 2)])
@pytest.mark.parametrize("out,inner", [(200, 320), (200, 1000), (65, 33)])
def test_library_rows_that_share_an_input_without_matrix_numbers(n_rows, per_input, out, inner):
    """`experts` may be null with any `per_input`: row r is x[r / per_input] times the one matrix.  Behind x's
    own rows lie NaN that no result may see; one row of x needs no stride."""
    L = _lib.load()
    m = neuzip.MX4Manager()
    w = rand(210, out, inner, scale=0.1)
    h = m.write(w.cuda())
    inputs = n_rows // per_input
    x = rand(211, inputs, inner)
    held = torch.full((inputs + 64, inner), float("nan"), dtype=torch.bfloat16, device="cuda")
    held[:inputs] = x.cuda()
    need = int(L.nz_mx4_linear_workspace_bytes(1, out, inner, n_rows, 0))
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    want, bound = mx4ref.product(x, w)
    for stride in (inner,) if inputs > 1 else (inner, 0):
        y = torch.empty(n_rows, out, dtype=torch.bfloat16, device="cuda")
        _lib.check(L.nz_mx4_linear(m._be.entry(h).packed.data_ptr(), 1, out, inner, _lib.NZ_DTYPE_BF16, held.data_ptr(),
                                   stride, n_rows, per_input, None, None, y.data_ptr(), ws.data_ptr(), need,
                                   status.data_ptr(), torch.cuda.current_stream().cuda_stream))
        mx4ref.check(y, want.repeat_interleave(per_input, 0), bound.repeat_interleave(per_input, 0))
    assert status.item() == 0
