"""4-bit matrices at the ends of what they hold and in the calls that are seldom made (kernels/mxfp4.py): scales near the end of the 32-bit range, results
that are not finite behind an activation, more rows than a launch's grid has along y, operands that only some kernels take, every split and tile."""
import pytest
import torch

from plain import mxfp4_plain as plain
from test_mxfp4_gpu import DEV, HALF_STEP, TYPES, _check, _matrix, _sum_bound, mx, ops

pytestmark = pytest.mark.gpu


def _scaled_matrix(rows, k, scale, seed):
    """A matrix of random codes under the given scale bytes [rows, blocks], and its values."""
    code = torch.randint(0, 16, (rows, scale.shape[1], 32), generator=torch.Generator().manual_seed(seed), dtype=torch.uint8)
    code.view(rows, -1)[:, k:] = 0
    w = mx().Mxfp4Matrix(plain.pack(code).to(DEV), scale.to(torch.uint8).to(DEV), k)
    return w, plain.values(code, scale, k).to(DEV)


# ---- scales near the end of the 32-bit range -----------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [1, 8, 9, 16, 33, 200])
@pytest.mark.parametrize("low,high,shift", [(200, 239, 0), (0, 245, -20), (232, 252, -100), (100, 250, -60)])
def test_high_scales(low, high, shift, M, dtype):
    """Scale bytes up to 252 under activations that keep the results in 32 bits: no step on the way leaves them either.  Every kernel, both kinds of
    activations, plain and gated."""
    if dtype is torch.float16 and shift < -24:
        pytest.skip("float16 has no such activations")
    m = mx()
    N, K = 140, 608
    g = torch.Generator().manual_seed(M + high)
    w, wv = _scaled_matrix(N, K, torch.randint(low, high + 1, (N, K // 32), generator=g), M)
    a = (torch.randn(M, K, generator=g) * 2.0 ** shift).to(dtype).to(DEV)
    for x, av in ((a, a.double()), (m.quantize_mxfp4(a), plain.rounded(a))):
        exact, bound = av @ wv.t(), _sum_bound(av, wv) + K * 2.0 ** -126                # products below 2^-126 may be lost in 32 bits
        assert float(exact.abs().max()) < 2.0 ** 127
        out = torch.empty(M, N, device=DEV)
        m.gemm_mxfp4(x, w, out)
        ops().raise_on_device_error()
        _check(out, exact, bound, torch.float32)
        if shift > -100:                                   # gate times up, each of 2^66 and more, would leave 32 bits
            continue
        gate, up = exact[:, :N // 2].clamp_min(0), exact[:, N // 2:]
        bg, bu = bound[:, :N // 2], bound[:, N // 2:]
        out = torch.empty(M, N // 2, device=DEV)
        m.gated_gemm_mxfp4(x, w, out, activation="relu")
        ops().raise_on_device_error()
        _check(out, gate * up, bg * up.abs() + gate * bu + bg * bu + 2.0 ** -23 * (gate * up).abs(), torch.float32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M", [1, 8, 9, 200])
def test_low_scales_beside_high_ones(M, dtype):
    """Blocks of the smallest scales between blocks of the largest, whose activations are zero: what they give keeps its bits."""
    m = mx()
    N, K = 70, 640
    g = torch.Generator().manual_seed(M)
    scale = torch.randint(229, 241, (N, K // 32), generator=g)
    scale[:, 1::2] = torch.randint(0, 12, (N, K // 64), generator=g)
    w, wv = _scaled_matrix(N, K, scale, M)
    a = torch.randn(M, K, generator=g) * 2.0 ** 100
    a.view(M, -1, 2, 32)[:, :, 0] = 0
    a = a.to(dtype).to(DEV)
    for x, av in ((a, a.double()), (m.quantize_mxfp4(a), plain.rounded(a))):
        out = torch.empty(M, N, device=DEV)
        m.gemm_mxfp4(x, w, out)
        ops().raise_on_device_error()
        _check(out, av @ wv.t(), _sum_bound(av, wv), torch.float32)
