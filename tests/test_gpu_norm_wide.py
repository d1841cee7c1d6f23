"""Layer norm of rows whose distances from the mean have squares past fp32: the definition in
64 bits, in the bounds of the other layer norm tests (their floor of 1e-30 left out: these
rows' dx is as small). Sums of a row stay below fp32's end."""

import math

import pytest
import torch
from test_gpu_norm import _check, _definition, _inputs, _run

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size", [1e17, 3e19, 1e25, 1e33])
@pytest.mark.parametrize("rows, d", [(5, 2), (300, 40), (37, 100), (70, 512), (33, 768), (9, 1000), (300, 2048), (20, 4097),
                                     (7, 8192), (3, 16384), (3, 16385), (2, 20000)])
def test_wide_rows(device, dtype, size, rows, d):
    x, dy, w, b = _inputs(device, (rows, d), dtype, seed=d, spread=size)
    x[rows // 2] = _inputs(device, (1, d), dtype, seed=1)[0][0]  # an ordinary row between them
    val, tol = _definition(x, dy, w, b, 1e-5)
    tol = [t - 1e-30 + 1e-42 for t in tol]
    got = _run(x, dy, w, b)
    _check(got, val, tol)
    assert (got[0].float().std(-1) > 0.3).all()  # the rows are normed, not emptied
    for p, q in zip(got, _run(x, dy, w, b)):
        assert torch.equal(p, q)


def test_rows_without_a_mean_stay_not_finite(device):
    x, dy, w, b = _inputs(device, (6, 300), F32, seed=3, spread=1e19)
    x[1, 7], x[2, 9], x[3] = math.inf, math.nan, 3e38
    y = _run(x, dy, w, b)[0]
    assert torch.isnan(y[1]).all() and torch.isnan(y[2]).all() and not torch.isfinite(y[3]).any()
    assert torch.isfinite(y[[0, 4, 5]]).all()
