"""4-bit matrices on the GPU against the definition in 64 bits (kernels/mxfp4.py)."""
import pytest
import torch

from plain import mxfp4_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
SMALLEST = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}     # half of the smallest step of all


def mx():
    from transformers_neuronx_b200.kernels import mxfp4
    return mxfp4


def ops():
    from transformers_neuronx_b200.kernels import ops as o
    return o


def _same(x, y):
    return torch.equal(x.isnan(), y.isnan()) and torch.equal(x.nan_to_num(0.0), y.nan_to_num(0.0)) and torch.equal(x.isinf(), y.isinf())


def _wide(rows, k, dtype, seed, spread=40.0):
    """Values over `spread` powers of two, between blocks and within them, whole blocks of zeros, ties."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=g)
    x = x * torch.exp2((torch.rand(rows, k, generator=g) - 0.5) * 6)
    x = x * torch.exp2(torch.round((torch.rand(rows, -(-k // 32), generator=g) - 0.5) * spread)).repeat_interleave(32, 1)[:, :k]
    ties = torch.tensor([0.25, -0.75, 1.25, 1.75, -2.5, 3.5, 5.0, 6.0, -0.0, 0.5, 7.0, 4.0])
    for r in range(0, rows, 3):
        n = min(k, 12)
        x[r, :n] = ties[:n]
    x[rows // 2, 32:64] = 0
    return x.to(dtype).to(DEV)


# one value, short last blocks, one block, rows that nothing divides, many blocks a row, many rows
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k,pad", [(1, 1, 0), (1, 31, 0), (1, 32, 0), (3, 33, 0), (7, 96, 8), (5, 100, 3), (2, 4096, 0), (129, 264, 0), (1000, 160, 0), (70000, 64, 0)])
def test_quantize(rows, k, pad, dtype):
    m = mx()
    x = _wide(rows, k + pad, dtype, rows + k)[:, :k]
    got = m.quantize_mxfp4(x)
    code, scale = plain.quantize(x)
    assert torch.equal(got.scales, scale) and torch.equal(got.codes, plain.pack(code))
    want = plain.values(code, scale, k)
    for t in TYPES:
        back = m.dequantize_mxfp4(got, t)
        assert back.dtype == t and back.shape == x.shape
        assert _same(back, want.to(t))                              # one rounding at most, and none but in float16
    out = torch.full((rows, k + 5), 7.0, device=DEV, dtype=dtype)
    m.dequantize_mxfp4(got, out=out[:, 2:2 + k])
    assert _same(out[:, 2:2 + k], want.to(dtype)) and bool((out[:, :2] == 7).all()) and bool((out[:, 2 + k:] == 7).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_extremes(dtype):
    """The type's largest and smallest numbers, infinities, NaN: a block that is not finite is NaN, its neighbours are whole."""
    m = mx()
    top = torch.finfo(dtype).max
    x = torch.zeros(6, 128, dtype=dtype)
    x[0, 5], x[0, 40] = top, -top
    x[1, 0], x[1, 33] = torch.finfo(dtype).smallest_normal, -torch.finfo(dtype).smallest_normal / 4
    x[2, 3], x[2, 4], x[2, 70] = float("inf"), 1.0, 3.0
    x[3, 31], x[3, 32] = float("nan"), 2.0
    x[4, 64] = float("-inf")
    x[5] = -0.0
    x = x.to(DEV)
    got = m.quantize_mxfp4(x)
    code, scale = plain.quantize(x)
    assert torch.equal(got.scales, scale) and torch.equal(got.codes, plain.pack(code))
    for t in TYPES:
        back = m.dequantize_mxfp4(got, t)
        assert torch.equal(back.isnan(), plain.values(code, scale, 128).isnan())
        if t != torch.float16:
            assert torch.equal(back.nan_to_num(0, 5, -5), plain.values(code, scale, 128).to(t).nan_to_num(0, 5, -5))


def test_every_scale_and_code():
    """All 16 codes under all 256 scales, as a checkpoint may hold them."""
    m = mx()
    code = torch.arange(16, dtype=torch.uint8).repeat(2).view(1, 1, 32).expand(256, 1, 32).contiguous().to(DEV)
    scale = torch.arange(256, dtype=torch.uint8).view(256, 1).to(DEV)
    w = m.Mxfp4Matrix(plain.pack(code), scale)
    want = plain.values(code, scale, 32)
    for t in (torch.float32, torch.bfloat16):
        got = m.dequantize_mxfp4(w, t)
        assert torch.equal(got.nan_to_num(0, 5, -5), want.to(t).nan_to_num(0, 5, -5)) and torch.equal(got.isnan(), want.isnan())


def _matrix(rows, k, seed, spread=8.0):
    """A 4-bit matrix of random codes whose scales lie `spread` powers of two apart, and its values."""
    g = torch.Generator().manual_seed(seed)
    blocks = -(-k // 32)
    code = torch.randint(0, 16, (rows, blocks, 32), generator=g, dtype=torch.uint8)
    code.view(rows, -1)[:, k:] = 0
    scale = (127 - 6 + torch.round((torch.rand(rows, blocks, generator=g) - 0.5) * spread)).to(torch.uint8)
    w = mx().Mxfp4Matrix(plain.pack(code).to(DEV), scale.to(DEV), k)
    return w, plain.values(code, scale, k).to(DEV)


def _sum_bound(a, w):
    """How far 32-bit sums may be off: a tensor-core accumulator cuts off at most 2^-22 of the sum of the products' sizes an addition, of
    which there is one for 16 columns at the most often; sums of parts and the rest round by 2^-24 a step, 64 steps at most."""
    size = a.abs() @ w.abs().t()
    return (-(-a.shape[1] // 16) * 2.0 ** -22 + 64 * 2.0 ** -24) * size


def _check(got, want, bound, dtype):
    """`bound` in the sums plus half a step of the result's type."""
    allowed = bound + HALF_STEP[dtype] * want.abs() * (1 + 2.0 ** -7) + SMALLEST[dtype]
    off = (got.double() - want).abs() - allowed
    assert bool((off <= 0).all()), float(off.max())


# one token to more than a tile, features below and above tiles of 64, 128 and 256, K of one block to many, odd sizes, short last blocks
SHAPES = [(1, 1, 32), (1, 128, 256), (1, 300, 96), (2, 64, 4096), (3, 1000, 1056), (5, 257, 20480), (8, 4096, 512), (13, 130, 2080), (16, 768, 768),
          (17, 200, 64), (33, 129, 288), (64, 2048, 1024), (100, 511, 320), (129, 640, 256), (200, 1030, 2080), (257, 136, 544), (300, 384, 100), (520, 2050, 1000)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gemm(M, N, K, dtype):
    m = mx()
    w, wv = _matrix(N, K, M + N + K)
    g = torch.Generator().manual_seed(K)
    a = torch.randn(M, K, generator=g).to(dtype).to(DEV)
    bias, res = torch.randn(N, generator=g).to(DEV), torch.randn(M, N, generator=g).to(DEV)
    av = a.double()
    exact, bound = av @ wv.t(), _sum_bound(av, wv)
    out = torch.full((M, N), float("nan"), device=DEV, dtype=dtype)
    assert m.gemm_mxfp4(a, w, out) is out
    ops().raise_on_device_error()
    _check(out, exact, bound, dtype)
    joined = res.clone()                                             # into the stream itself
    m.gemm_mxfp4(a, w, joined, bias=bias, residual=joined, activation="relu")
    want = (exact + bias.double()).clamp_min(0) + res.double()
    _check(joined, want, bound + 2.0 ** -23 * (exact.abs() + bias.double().abs()), torch.float32)
    again = res.clone()
    m.gemm_mxfp4(a, w, again, bias=bias, residual=again, activation="relu")
    assert torch.equal(again, joined)                                # the order of sums is fixed


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gemm_both_in_4_bits(M, N, K, dtype):
    m = mx()
    w, wv = _matrix(N, K, M + N + K)
    g = torch.Generator().manual_seed(K)
    a = torch.randn(M, K, generator=g).to(DEV)
    bias, res = torch.randn(N, generator=g).to(DEV), torch.randn(M, N, generator=g).to(DEV)
    q, av = m.quantize_mxfp4(a), plain.rounded(a)
    exact, bound = av @ wv.t(), _sum_bound(av, wv)
    out = torch.full((M, N), float("nan"), device=DEV, dtype=dtype)
    m.gemm_mxfp4(q, w, out, bias=bias)
    ops().raise_on_device_error()
    _check(out, exact + bias.double(), bound + 2.0 ** -23 * (exact.abs() + bias.double().abs()), dtype)
    joined = res.clone()
    m.gemm_mxfp4(q, w, joined, residual=joined)
    _check(joined, exact + res.double(), bound + 2.0 ** -23 * exact.abs(), torch.float32)


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,F,K,act", [(1, 64, 256, "silu"), (1, 1, 32, "relu"), (2, 257, 512, "gelu_new"), (7, 1000, 1056, "silu"), (16, 512, 4096, "gelu"),
                                       (40, 130, 96, "none"), (130, 72, 320, "silu"), (300, 520, 544, "relu2"), (515, 64, 1000, "silu")])
def test_gated(M, F, K, act, dtype, quantized):
    m = mx()
    w, wv = _matrix(2 * F, K, M + F + K)
    g = torch.Generator().manual_seed(K)
    a = torch.randn(M, K, generator=g).to(dtype).to(DEV)
    bias = torch.randn(2 * F, generator=g).to(DEV)
    av = plain.rounded(a) if quantized else a.double()
    both = av @ wv.t() + bias.double()
    off = _sum_bound(av, wv) + 2.0 ** -23 * both.abs()
    gate, up = plain.activation(both[:, :F], act), both[:, F:]
    # the activations' slopes are at most 1.13 (relu2: 2 |x|), each is computed within 2^-18 of its argument's size
    slope = 2 * (both[:, :F].abs() + off[:, :F]) if act == "relu2" else 1.13
    off_gate = slope * off[:, :F] + 2.0 ** -18 * both[:, :F].abs()
    bound = off_gate * up.abs() + gate.abs() * off[:, F:] + off_gate * off[:, F:] + 2.0 ** -23 * (gate * up).abs()
    out = torch.full((M, F), float("nan"), device=DEV, dtype=dtype)
    assert m.gated_gemm_mxfp4(m.quantize_mxfp4(a) if quantized else a, w, out, bias=bias, activation=act) is out
    ops().raise_on_device_error()
    _check(out, gate * up, bound, dtype)


@pytest.mark.parametrize("act", ["none", "relu", "relu2", "silu", "sigmoid", "gelu", "gelu_new"])
@pytest.mark.parametrize("M", [3, 150])
def test_activations(M, act):
    m = mx()
    w, wv = _matrix(192, 256, M, spread=2.0)
    a = torch.randn(M, 256, generator=torch.Generator().manual_seed(M)).bfloat16().to(DEV)
    exact, bound = a.double() @ wv.t(), _sum_bound(a.double(), wv)
    slope = 2 * (exact.abs() + bound) if act == "relu2" else 1.13
    out = torch.empty(M, 192, device=DEV)
    m.gemm_mxfp4(a, w, out, activation=act)
    _check(out, plain.activation(exact, act), slope * bound + 2.0 ** -18 * (exact.abs() + 1), torch.float32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M", [1, 4, 40, 200])
def test_pitches_and_slices(M, dtype):
    """Activations and results that are columns of wider buffers, matrices that are rows of larger ones, bases that no tensor map takes;
    what lies beside the result stays as it was."""
    m = mx()
    N, K = 264, 512
    big, bigv = _matrix(2 * N + 1, K, M)
    g = torch.Generator().manual_seed(M)
    for row, a_off, o_off in ((0, 0, 0), (N, 8, 8), (1, 3, 5)):
        w = m.Mxfp4Matrix(big.codes[row:row + N], big.scales[row:row + N])
        wide = torch.randn(M, K + 24, generator=g).to(dtype).to(DEV)
        a = wide[:, a_off:a_off + K]
        buf = torch.full((M, N + 16), 7.0, device=DEV, dtype=dtype)
        m.gemm_mxfp4(a, w, buf[:, o_off:o_off + N])
        ops().raise_on_device_error()
        wv = bigv[row:row + N]
        _check(buf[:, o_off:o_off + N], a.double() @ wv.t(), _sum_bound(a.double(), wv), dtype)
        assert bool((buf[:, :o_off] == 7).all()) and bool((buf[:, o_off + N:] == 7).all())
    shifted = torch.empty(N * K // 2 + 16, dtype=torch.uint8, device=DEV)          # codes that begin at an odd address
    shifted[3:3 + N * K // 2] = big.codes[:N].flatten()
    w = m.Mxfp4Matrix(shifted[3:3 + N * K // 2].view(N, K // 2), big.scales[:N])
    a = torch.randn(M, K, generator=g).to(dtype).to(DEV)
    out = torch.empty(M, N, device=DEV, dtype=dtype)
    m.gemm_mxfp4(a, w, out)
    _check(out, a.double() @ bigv[:N].t(), _sum_bound(a.double(), bigv[:N]), dtype)
    q = m.quantize_mxfp4(a)
    m.gemm_mxfp4(q, w, out)
    av = plain.rounded(a)
    _check(out, av @ bigv[:N].t(), _sum_bound(av, bigv[:N]), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [1, 12, 70, 300])
@pytest.mark.parametrize("low,high", [(127 - 100, 127 + 20), (127 - 30, 127 + 30), (0, 10), (250 - 127, 127)])
def test_scales_far_apart(M, low, high, dtype):
    """Blocks whose scales lie up to 120 powers of two apart in one row: every term counts with the size it has."""
    m = mx()
    g = torch.Generator().manual_seed(M + low)
    N, K = 140, 512
    code = torch.randint(0, 16, (N, K // 32, 32), generator=g, dtype=torch.uint8)
    scale = torch.randint(low, high + 1, (N, K // 32), generator=g).to(torch.uint8)
    w, wv = m.Mxfp4Matrix(plain.pack(code).to(DEV), scale.to(DEV)), plain.values(code, scale, K).to(DEV)
    a = torch.randn(M, K, generator=g).to(dtype).to(DEV)
    out = torch.empty(M, N, device=DEV)
    m.gemm_mxfp4(a, w, out)
    ops().raise_on_device_error()
    # products below 2^-126 may be lost in 32 bits
    _check(out, a.double() @ wv.t(), _sum_bound(a.double(), wv) + K * 2.0 ** -126, torch.float32)
    # rows of the matrix in which only the small blocks meet activations that are not zero
    for r in range(K // 32):
        b = torch.zeros_like(a)
        b[:, 32 * r:32 * r + 32] = a[:, 32 * r:32 * r + 32]
        if r % 5 == 0:
            m.gemm_mxfp4(b, w, out)
            top = a.double().abs().sum(1, keepdim=True) * wv.abs().amax(1)         # a row keeps 2^-36 of its largest block at least
            _check(out, b.double() @ wv.t(), _sum_bound(b.double(), wv) + K * 2.0 ** -126 + (2.0 ** -36 * top if dtype == torch.float16 else 0), torch.float32)


@pytest.mark.parametrize("M", [1, 20, 200])
@pytest.mark.parametrize("quantized", [False, True])
def test_not_finite(M, quantized):
    """A NaN block of the matrix makes its feature NaN and no other; an infinite activation its token."""
    m = mx()
    w, wv = _matrix(150, 320, 3)
    w.scales[7, 4] = 255
    a = torch.randn(M, 320, generator=torch.Generator().manual_seed(M)).bfloat16().to(DEV)
    out = torch.zeros(M, 150, device=DEV)
    m.gemm_mxfp4(m.quantize_mxfp4(a) if quantized else a, w, out)
    assert bool(out[:, 7].isnan().all()) and int(out.isnan().sum()) == M
    a[0, 11] = float("inf")
    w.scales[7, 4] = 120
    m.gemm_mxfp4(m.quantize_mxfp4(a) if quantized else a, w, out)
    assert not bool(out[0].isfinite().any()) and bool(out[1:].isfinite().all())


def test_nothing_to_do():
    m = mx()
    w, _ = _matrix(64, 96, 1)
    assert m.gemm_mxfp4(torch.empty(0, 96, device=DEV), w, torch.empty(0, 64, device=DEV)).shape == (0, 64)
    assert m.quantize_mxfp4(torch.empty(0, 96, device=DEV)).shape == (0, 96)
    assert m.dequantize_mxfp4(m.quantize_mxfp4(torch.empty(0, 96, device=DEV))).shape == (0, 96)


def test_refusals():
    m = mx()
    w, _ = _matrix(64, 96, 1)
    a, out = torch.zeros(4, 96, device=DEV), torch.zeros(4, 64, device=DEV)
    bad = [lambda: m.gemm_mxfp4(a[:, :64], w, out), lambda: m.gemm_mxfp4(a, w, out[:, :63]), lambda: m.gemm_mxfp4(a[:3], w, out),
           lambda: m.gemm_mxfp4(a.double(), w, out), lambda: m.gemm_mxfp4(a.half(), w, out.bfloat16()), lambda: m.gemm_mxfp4(a, w, out.t()),
           lambda: m.gemm_mxfp4(a, w, out, bias=torch.zeros(63, device=DEV)), lambda: m.gemm_mxfp4(a, w, out, bias=torch.zeros(64)),
           lambda: m.gemm_mxfp4(a, w, out.bfloat16(), residual=out), lambda: m.gemm_mxfp4(a, w, out, residual=torch.zeros(4, 65, device=DEV)[:, :64]),
           lambda: m.gemm_mxfp4(a, w, out, activation="softplus"), lambda: m.gated_gemm_mxfp4(a, w, out), lambda: m.gemm_mxfp4(a.cpu(), w, out),
           lambda: m.quantize_mxfp4(a.t()[:, :3]), lambda: m.quantize_mxfp4(a, out=w), lambda: m.dequantize_mxfp4(w, torch.float64),
           lambda: m.dequantize_mxfp4(w, out=out), lambda: m.quantize_mxfp4(a[:, :0])]
    for i, call in enumerate(bad):
        with pytest.raises(m.KernelError):
            call()
            pytest.fail(f"call {i} was taken")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(700, 9001, 96), (1040, 6000, 288), (385, 20000, 64), (2048, 4100, 1312), (150, 60000, 32)])
def test_many_tiles(M, N, K, dtype):
    """Blocks that walk over several tiles: all kinds of operands, plain and gated, every element."""
    m = mx()
    w, wv = _matrix(N, K, M + N + K)
    g = torch.Generator().manual_seed(K)
    a = torch.randn(M, K, generator=g).to(dtype).to(DEV)
    bias = torch.randn(N, generator=g).to(DEV)
    for x, av in ((a, a.double()), (m.quantize_mxfp4(a), plain.rounded(a))):
        exact, bound = av @ wv.t() + bias.double(), _sum_bound(av, wv)
        bound = bound + 2.0 ** -23 * (exact.abs() + bias.double().abs())
        out = torch.full((M, N), float("nan"), device=DEV, dtype=dtype)
        m.gemm_mxfp4(x, w, out, bias=bias)
        ops().raise_on_device_error()
        _check(out, exact, bound, dtype)
        if N % 2 == 0:
            F = N // 2
            out = torch.full((M, F), float("nan"), device=DEV, dtype=dtype)
            m.gated_gemm_mxfp4(x, w, out, bias=bias, activation="relu")
            gate, up = exact[:, :F].clamp_min(0), exact[:, F:]
            both = bound[:, :F] * up.abs() + gate * bound[:, F:] + bound[:, :F] * bound[:, F:] + 2.0 ** -23 * (gate * up).abs()
            _check(out, gate * up, both, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", [(64, 256, 20480), (200, 300, 20480), (300, 512, 6144)])
def test_long_sums_in_32_bits(M, N, K, dtype):
    """Long sums into 32-bit results: random operands, whose additions round either way, lose less than 2^-20 of the result."""
    from transformers_neuronx_b200.kernels import build
    m = mx()
    assert build.load("gemm_mxfp4", dtype).tnx_gemm_mxfp4_chain() == m.CHAIN
    w, wv = _matrix(N, K, M + K, spread=2.0)
    a = torch.randn(M, K, generator=torch.Generator().manual_seed(K)).to(dtype).to(DEV)
    out = torch.empty(M, N, device=DEV)
    m.gemm_mxfp4(a, w, out)
    ops().raise_on_device_error()
    want = a.double() @ wv.t()
    assert float((out.double() - want).norm() / want.norm()) <= 2.0 ** -20
