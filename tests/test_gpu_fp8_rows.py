"""Memory behind the last column of 8-bit rows, on a real MI355X."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [1, 5, 100, 129, 190, 251, 500, 1027, 2049, 4100, 8201])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_writes_zeros_up_to_the_next_multiple_of_eight(dev, d, residual):
    """Also in rows without a finite norm: a NaN, an infinity, zeros with eps = 0.  What lies further is left alone."""
    from src import _native as N
    T, ld = 5, -(-d // 8) * 8 + 24
    x = torch.randn(T, d, device=dev)
    x[1, d // 2] = math.nan
    x[2, d - 1] = math.inf
    x[3] = 0
    res = torch.zeros(T, d, device=dev) if residual else None
    out = torch.empty(T, d, device=dev)
    w = torch.ones(d, device=dev)
    q = torch.full((T + 1, ld), 0x55, dtype=torch.uint8, device=dev)
    nb = -(-d // 128)
    scale = torch.full((T + 1, nb + 3), 0x33, dtype=torch.uint8, device=dev)
    rc = N.lib().ldm_rmsnorm_fp8(x.data_ptr(), N.F32, d, res.data_ptr() if residual else None, N.F32, d, w.data_ptr(), T, d, 0.0,
                                 out.data_ptr(), q.data_ptr(), ld, scale.data_ptr(), nb + 3, N.stream())
    torch.cuda.synchronize()
    assert rc == 0
    up = -(-d // 8) * 8
    assert bool((q[:T, d:up] == 0).all())
    assert bool((q[:T, up:] == 0x55).all()) and bool((q[T] == 0x55).all())
    assert bool((scale[:T, nb:] == 0x33).all()) and bool((scale[T] == 0x33).all())
    v = q[:T, :d].contiguous().view(torch.float8_e4m3fn).float()
    assert bool(v[1].isnan().all()) and bool(v[3].isnan().all()) and not bool(v[[0, 4]].isnan().any())


@pytest.mark.parametrize("swiglu", [0, 1])
@pytest.mark.parametrize("d", [1, 5, 100, 129, 1027])
def test_rows_write_zeros_up_to_the_next_multiple_of_eight(dev, d, swiglu):
    from src import _native as N
    T, ld, nb, up = 4, -(-d // 8) * 8 + 24, -(-d // 128), -(-d // 8) * 8
    x = torch.randn(T, d * (1 + swiglu), device=dev)
    x[1] = math.nan
    x[2] = math.inf
    q = torch.full((T + 1, ld), 0x55, dtype=torch.uint8, device=dev)
    scale = torch.full((T + 1, nb + 3), 0x33, dtype=torch.uint8, device=dev)
    rc = N.lib().ldm_quant_fp8(x.data_ptr(), N.F32, x.shape[1], T, d, swiglu, q.data_ptr(), ld, scale.data_ptr(), nb + 3, N.stream())
    torch.cuda.synchronize()
    assert rc == 0 and bool((q[:T, d:up] == 0).all()) and bool((q[:T, up:] == 0x55).all()) and bool((q[T] == 0x55).all())
    assert bool((scale[:T, nb:] == 0x33).all()) and bool((scale[T] == 0x33).all())
