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


# ---- sums that are not finite, or far below zero, behind an activation ---------------------------------------------
SUMS = [float("nan"), float("-inf"), float("inf"), -3e38, -1e30, -2e4, -200.0, -70.0, -20.0, -5.0, -0.5, 0.0, 0.5, 5.0, 20.0, 3e4, 1e30, 3e38]
ACTS = ["none", "relu", "relu2", "silu", "sigmoid", "gelu", "gelu_new"]


def _sources(m, M, K, dtype, seed):
    """The kinds of activations that different kernels take: `dtype`, rows that no tensor map takes, 4 bits."""
    a = torch.randn(M, K + 3, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)
    return [a[:, 3:], a[:, :K].contiguous(), m.quantize_mxfp4(a[:, :K])]


def _check_sums(got, x, act, dtype):
    """got = act(x) in `dtype`, x exact sums.  32-bit results: exp, tanh and erf within two units in the last place, an addition and a division (3 * 2^-23 in
    all), 16-bit ones: an exp(x) with 2 + 1.2 |x| units, |x| <= 90.  Where 1 + tanh or 1 + erf nearly cancel, 2^-22 of the argument's size is left over (it
    is whole beyond 100).  exp leaves its range at 88.7: 2^-120."""
    want = plain.activation(x.double(), act).to(torch.float32).double()
    there = want.to(dtype)
    assert torch.equal(got.isnan(), there.isnan()), (got, there)
    assert torch.equal(got.isinf(), there.isinf()) and torch.equal(got[there.isinf()] > 0, there[there.isinf()] > 0), (got, there)
    rel = 2.0 ** -21 if dtype is torch.float32 else HALF_STEP[dtype] * (1 + 2.0 ** -7) + 2.0 ** -16
    off = rel * want.abs() + 2.0 ** -120 + (2.0 ** -25 if dtype is torch.float16 else 0.0)
    if act in ("gelu", "gelu_new"):
        off = off + 2.0 ** -22 * x.double().abs().clamp_max(100)
    fine = there.isfinite()
    bad = ((got.double() - want).abs() > off) & fine
    assert not bool(bad.any()), (act, x[bad], got[bad], want[bad])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [2, 20, 200])
@pytest.mark.parametrize("act", ACTS)
def test_activations_of_given_sums(act, M, dtype):
    """Zero products, so that the bias is the sum: infinities, NaN and numbers of every size through every activation."""
    m = mx()
    K = 96
    x = torch.tensor(SUMS * 8, device=DEV)
    F = len(x)
    w = m.Mxfp4Matrix(torch.zeros(2 * F, K // 2, dtype=torch.uint8, device=DEV), torch.full((2 * F, K // 32), 127, dtype=torch.uint8, device=DEV))
    half = m.Mxfp4Matrix(w.codes[:F], w.scales[:F])
    for a in _sources(m, M, K, dtype, M):
        out = torch.full((M, F), 7.0, device=DEV, dtype=dtype)
        m.gemm_mxfp4(a, half, out, bias=x, activation=act)
        ops().raise_on_device_error()
        _check_sums(out, x.expand(M, F), act, dtype)
        out = torch.full((M, F), 7.0, device=DEV, dtype=dtype)
        m.gated_gemm_mxfp4(a, w, out, bias=torch.cat((x, torch.ones_like(x))), activation=act)
        ops().raise_on_device_error()
        _check_sums(out, x.expand(M, F), act, dtype)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M", [1, 9, 200])
def test_blocks_that_are_not_a_number_behind_activations(M, act):
    """A block of scale byte 255 makes its feature NaN whatever the activation, in the gate's rows and in the up rows, and no other."""
    m = mx()
    K, F = 320, 90
    for row, feature in ((7, 7), (F + 11, 11)):
        w, _ = _matrix(2 * F, K, 3)
        w.scales[row, 4] = 255
        for a in _sources(m, M, K, torch.bfloat16, M):
            out = torch.zeros(M, 2 * F, device=DEV)
            m.gemm_mxfp4(a, w, out, activation=act)
            assert bool(out[:, row].isnan().all()) and int(out.isnan().sum()) == M
            out = torch.zeros(M, F, device=DEV, dtype=torch.bfloat16)
            m.gated_gemm_mxfp4(a, w, out, activation=act)
            assert bool(out[:, feature].isnan().all()) and int(out.isnan().sum()) == M
    ops().raise_on_device_error()


# ---- more rows of W than 65,535 tiles ------------------------------------------------------------------------------
@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("M", [1, 16, 64, 130])
def test_more_than_65535_tiles(M, quantized):
    m = mx()
    K, N = 32, 65535 * 128 + 200
    g = torch.Generator(device=DEV).manual_seed(M)
    codes = torch.empty(N, 16, device=DEV, dtype=torch.uint8).random_(0, 256, generator=g)
    scales = torch.empty(N, 1, device=DEV, dtype=torch.uint8).random_(118, 126, generator=g)
    w = m.Mxfp4Matrix(codes, scales)
    a = torch.randn(M, K, generator=g, device=DEV).bfloat16()
    x, av = (m.quantize_mxfp4(a), plain.rounded(a)) if quantized else (a, a.double())

    def values(rows):
        return m.dequantize_mxfp4(m.Mxfp4Matrix(codes[rows].contiguous(), scales[rows].contiguous()), torch.float32).double()
    out = torch.full((M, N), float("nan"), device=DEV, dtype=torch.bfloat16)
    m.gemm_mxfp4(x, w, out)
    ops().raise_on_device_error()
    at = torch.tensor([0, 127, 128, 65534 * 128, 65535 * 128 - 1, 65535 * 128, 65535 * 128 + 1, N - 1], device=DEV)
    wv = values(at)
    _check(out[:, at], av @ wv.t(), _sum_bound(av, wv), torch.bfloat16)
    assert not bool(out.isnan().any())
    F = N // 2                                             # more than 65,535 tiles of 64 features
    out = torch.full((M, F), float("nan"), device=DEV, dtype=torch.bfloat16)
    m.gated_gemm_mxfp4(x, w, out, activation="relu")
    ops().raise_on_device_error()
    at = torch.tensor([0, 63, 64, 65534 * 64, 65535 * 64 - 1, 65535 * 64, F - 1], device=DEV)
    gv, uv = values(at), values(F + at)
    gate, up, bg, bu = (av @ gv.t()).clamp_min(0), av @ uv.t(), _sum_bound(av, gv), _sum_bound(av, uv)
    _check(out[:, at], gate * up, bg * up.abs() + gate * bu + bg * bu + 2.0 ** -23 * (gate * up).abs(), torch.bfloat16)
    assert not bool(out.isnan().any())


def test_more_than_65535_tiles_of_long_rows():
    """32-bit results of more than 5,120 columns: 130 tokens, whose K is split (22 GB of codes)."""
    m = mx()
    M, K, N = 130, 5152, 65535 * 128 + 200
    g = torch.Generator(device=DEV).manual_seed(1)
    codes = torch.empty(N, K // 2, device=DEV, dtype=torch.uint8).random_(0, 256, generator=g)
    scales = torch.empty(N, K // 32, device=DEV, dtype=torch.uint8).random_(118, 126, generator=g)
    a = torch.randn(M, K, generator=g, device=DEV).bfloat16()
    out = torch.full((M, N), float("nan"), device=DEV)
    m.gemm_mxfp4(a, m.Mxfp4Matrix(codes, scales), out)
    ops().raise_on_device_error()
    at = torch.tensor([0, 128, 65535 * 128 - 1, 65535 * 128, N - 1], device=DEV)
    wv = m.dequantize_mxfp4(m.Mxfp4Matrix(codes[at].contiguous(), scales[at].contiguous()), torch.float32).double()
    _check(out[:, at], a.double() @ wv.t(), _sum_bound(a.double(), wv), torch.float32)
    del codes, scales, out
    torch.cuda.empty_cache()


# ---- which build of the kernels ------------------------------------------------------------------------------------
def _loaded_flavours(m, monkeypatch, run):
    """The flavours in which run() asks for this family's libraries."""
    from transformers_neuronx_b200.kernels import build
    asked, load = set(), build.load

    def recording(name, dtype=None):
        if "mxfp4" in name:
            asked.add((name, build.flavour_of(dtype)))
        return load(name, dtype)
    with monkeypatch.context() as p:
        p.setattr(build, "load", recording)
        p.setattr(m, "_entries", {})
        p.setattr(m, "_tiles", {})
        run()
    return asked


@pytest.mark.parametrize("dtype,flavour", [(torch.float16, "f16"), (torch.bfloat16, "")])
@pytest.mark.parametrize("M", [1, 16, 200])
def test_flavour_of_4_bit_activations(M, dtype, flavour, monkeypatch):
    """Operands that came from one 16-bit type go to the kernels built for it, into 32 bits too, whichever of the two tells."""
    m = mx()
    x, w = torch.randn(M, 256, device=DEV).to(dtype), torch.randn(300, 256, device=DEV).to(dtype)
    out = torch.empty(M, 300, device=DEV)

    def run():
        q = m.quantize_mxfp4(w)
        m.gemm_mxfp4(m.quantize_mxfp4(x), q, out)
        m.gemm_mxfp4(m.quantize_mxfp4(x), m.Mxfp4Matrix(q.codes, q.scales), out)
        m.gemm_mxfp4(m.Mxfp4Matrix(*(lambda p: (p.codes, p.scales))(m.quantize_mxfp4(x))), q, out)
        m.gemm_mxfp4(m.quantize_mxfp4(x, out=m.quantize_mxfp4(x.clone())), q, out)
    assert {f for _, f in _loaded_flavours(m, monkeypatch, run)} == {flavour}


# ---- the slices of a product on the multiply-add units -------------------------------------------------------------
def test_most_tokens_of_one_column():
    """2^31 - 4,096 tokens of one value by a matrix of one row (4.3 GB each way): the slices' counter stays in its range."""
    m = mx()
    M = m.MOST
    w = m.Mxfp4Matrix(torch.tensor([[4] + [0] * 15], dtype=torch.uint8, device=DEV), torch.tensor([[127]], dtype=torch.uint8, device=DEV), 1)     # 2
    a = torch.ones(M, 1, device=DEV, dtype=torch.float16)
    a[-1] = 3
    a[M // 2] = 5
    out = torch.zeros(M, 1, device=DEV, dtype=torch.float16)
    m.gemm_mxfp4(a, w, out)
    ops().raise_on_device_error()
    assert float(out[-1]) == 6 and float(out[M // 2]) == 10
    out[-1] = out[M // 2] = 2
    for part in out.split(1 << 28):
        assert bool((part == 2).all())
    del a, out, part
    torch.cuda.empty_cache()


# ---- 4-bit activations that no tensor map takes --------------------------------------------------------------------
@pytest.mark.parametrize("M", [1, 8, 9, 16, 17])
@pytest.mark.parametrize("spread", [4.0, 60.0])
def test_4_bit_activations_off_16_bytes(M, spread):
    """Codes of the activations that begin four bytes into a buffer: the streaming kernel takes up to 16 tokens of them, the multiply-add units more."""
    m = mx()
    N, K = 150, 1000
    g = torch.Generator().manual_seed(M)
    w, wv = _matrix(N, K, M)
    a = torch.randn(M, K, generator=g) * torch.exp2(torch.round((torch.rand(M, 32, generator=g) - 0.5) * spread)).repeat_interleave(32, 1)[:, :K]
    q = m.quantize_mxfp4(a.to(DEV))
    n = q.codes.numel()
    buf = torch.zeros(n + 16, dtype=torch.uint8, device=DEV)
    buf[4:4 + n] = q.codes.flatten()
    x = m.Mxfp4Matrix(buf[4:4 + n].view(M, -1), q.scales, K)
    av = plain.rounded(a.to(DEV))
    # values below 2^-39 of the largest of the 256 around them are not told from zero by the streaming kernel
    pad = torch.nn.functional.pad(av.abs(), (0, -K % 256)).view(M, -1, 256).amax(-1)
    wide = torch.nn.functional.pad(wv.abs(), (0, -K % 256)).view(N, -1, 256).sum(-1)
    bound = _sum_bound(av, wv) + 2.0 ** -39 * (pad @ wide.t())
    out = torch.empty(M, N, device=DEV)
    m.gemm_mxfp4(x, w, out)
    ops().raise_on_device_error()
    _check(out, av @ wv.t(), bound, torch.float32)
    gate, up = (av @ wv[:75].t()).clamp_min(0), av @ wv[75:].t()
    out = torch.empty(M, 75, device=DEV)
    m.gated_gemm_mxfp4(x, w, out, activation="relu")
    ops().raise_on_device_error()
    bg, bu = bound[:, :75], bound[:, 75:]
    _check(out, gate * up, bg * up.abs() + gate * bu + bg * bu + 2.0 ** -23 * (gate * up).abs(), torch.float32)


# ---- every plan ----------------------------------------------------------------------------------------------------
def _force(library, dtype, name, *values):
    from transformers_neuronx_b200.kernels import build
    return getattr(build.load(library, dtype), name)(*values)


def _all_results(m, w, wv, x, av, bias, dtype):
    """The product and (an even number of rows) the gated one, checked."""
    N = w.rows
    exact, bound = av @ wv.t() + bias.double(), _sum_bound(av, wv)
    bound = bound + 2.0 ** -23 * (exact.abs() + bias.double().abs())
    out = torch.full((av.shape[0], N), float("nan"), device=DEV, dtype=dtype)
    m.gemm_mxfp4(x, w, out, bias=bias)
    ops().raise_on_device_error()
    _check(out, exact, bound, dtype)
    F = N // 2
    out = torch.full((av.shape[0], F), float("nan"), device=DEV, dtype=dtype)
    m.gated_gemm_mxfp4(x, w, out, bias=bias, activation="relu")
    ops().raise_on_device_error()
    gate, up, bg, bu = exact[:, :F].clamp_min(0), exact[:, F:], bound[:, :F], bound[:, F:]
    _check(out, gate * up, bg * up.abs() + gate * bu + bg * bu + 2.0 ** -23 * (gate * up).abs(), dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("splits", range(1, 9))
def test_every_split_and_width_of_a_tile(splits, dtype):
    m = mx()
    N, K = 266, (2 * splits - 1) * 256 - 160               # two boxes a part, the last one's ragged
    w, wv = _matrix(N, K, splits)
    g = torch.Generator().manual_seed(splits)
    bias = torch.randn(N, generator=g).to(DEV)
    try:
        for bn in (16, 32, 64, 128):
            assert _force("gemm_mxfp4", dtype, "tnx_gemm_mxfp4_force", bn, splits) == 0
            for M in (13, 117):
                a = torch.randn(M, K, generator=g).to(dtype).to(DEV)
                _all_results(m, w, wv, a, a.double(), bias, dtype)
                _all_results(m, w, wv, m.quantize_mxfp4(a), plain.rounded(a), bias, dtype)
    finally:
        _force("gemm_mxfp4", dtype, "tnx_gemm_mxfp4_force", 0, 0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bn", range(64, 193, 16))
def test_every_width_of_a_persistent_tile(bn, dtype, monkeypatch):
    m = mx()
    N, K = 1034, 544
    w, wv = _matrix(N, K, bn)
    g = torch.Generator().manual_seed(bn)
    bias = torch.randn(N, generator=g).to(DEV)
    monkeypatch.setattr(m, "_in_tiles", lambda *a: True)
    try:
        assert _force("gemm_mxfp4_tiles", dtype, "tnx_gemm_mxfp4_tiles_force", bn) == 0
        for M in (129, 1500):
            a = torch.randn(M, K, generator=g).to(dtype).to(DEV)
            _all_results(m, w, wv, a, a.double(), bias, dtype)
            _all_results(m, w, wv, m.quantize_mxfp4(a), plain.rounded(a), bias, dtype)
    finally:
        _force("gemm_mxfp4_tiles", dtype, "tnx_gemm_mxfp4_tiles_force", 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("splits", [1, 2, 4, 8])
def test_every_plan_of_streamed_products(splits, dtype):
    m = mx()
    N, K = 266, 4000
    w, wv = _matrix(N, K, splits)
    g = torch.Generator().manual_seed(splits)
    bias = torch.randn(N, generator=g).to(DEV)
    try:
        for wf in range(1, 16):
            assert _force("gemv_mxfp4", dtype, "tnx_gemv_mxfp4_force", wf, splits) == 0
            for M in (1, 7, 16) if dtype is torch.float32 else (1, 7):
                a = torch.randn(M, K, generator=g).to(dtype).to(DEV)
                _all_results(m, w, wv, a, a.double(), bias, dtype)
    finally:
        _force("gemv_mxfp4", dtype, "tnx_gemv_mxfp4_force", 0, 0)


def test_forced_plans_that_are_none_are_refused():
    for library, name, bad in (("gemm_mxfp4", "tnx_gemm_mxfp4_force", ((48, 0), (0, 9), (-16, 1))), ("gemm_mxfp4_tiles", "tnx_gemm_mxfp4_tiles_force", ((48,), (72,), (208,))),
                               ("gemv_mxfp4", "tnx_gemv_mxfp4_force", ((16, 1), (1, 3), (-1, 0)))):
        for values in bad:
            assert _force(library, torch.bfloat16, name, *values) != 0


# ---- long sums of two 4-bit operands -------------------------------------------------------------------------------
@pytest.mark.parametrize("M,N,K", [(16, 256, 20480), (64, 256, 65536), (200, 300, 20480), (300, 512, 65536)])
def test_long_sums_of_4_bit_activations(M, N, K):
    """One accumulator adds up all of K, 64 columns an addition: random operands whose scales spread over 2^8 lose less than 2^-20 of the result, as sums of
    16-bit activations do in chains of a quarter of that."""
    m = mx()
    w, wv = _matrix(N, K, M + K, spread=8.0)
    g = torch.Generator().manual_seed(K)
    a = torch.randn(M, K, generator=g) * torch.exp2(torch.round((torch.rand(M, K // 32, generator=g) - 0.5) * 8)).repeat_interleave(32, 1)
    a = a.bfloat16().to(DEV)
    out = torch.empty(M, N, device=DEV)
    m.gemm_mxfp4(m.quantize_mxfp4(a), w, out)
    ops().raise_on_device_error()
    want = plain.rounded(a) @ wv.t()
    assert float((out.double() - want).norm() / want.norm()) <= 2.0 ** -20
