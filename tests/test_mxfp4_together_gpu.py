"""4-bit matrices on the GPU: operators one behind another, on other streams, in captured graphs, on matrices of more than 4 GB, and the calls that are
easily got wrong (kernels/mxfp4.py)."""
import pytest
import torch

from plain import mxfp4_plain as plain
from test_mxfp4_gpu import DEV, _check, _matrix, _sum_bound, mx, ops

pytestmark = pytest.mark.gpu


def _feed_forward(m, x, gate_up, down, quantized, out):
    """A gated feed-forward's two products, the residual stream `out` [tokens, hidden] in 32 bits."""
    h = torch.empty(x.shape[0], gate_up.rows // 2, device=DEV, dtype=x.dtype)
    m.gated_gemm_mxfp4(m.quantize_mxfp4(x) if quantized else x, gate_up, h)
    m.gemm_mxfp4(m.quantize_mxfp4(h) if quantized else h, down, out, residual=out)
    return h


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens", [1, 12, 100, 700])
def test_feed_forward(tokens, dtype, quantized):
    """Each product against the definition on what it was given; again and again without a wait between the calls: the same bits."""
    m = mx()
    H, F = 416, 1000
    gate_up, guv = _matrix(2 * F, H, 5, 4.0)
    down, dv = _matrix(H, F, 6, 4.0)
    g = torch.Generator().manual_seed(tokens)
    x = torch.randn(tokens, H, generator=g).to(dtype).to(DEV)
    res = torch.randn(tokens, H, generator=g).to(DEV)
    out = res.clone()
    h = _feed_forward(m, x, gate_up, down, quantized, out)
    ops().raise_on_device_error()
    xv = plain.rounded(x) if quantized else x.double()
    gate, up = xv @ guv[:F].t(), xv @ guv[F:].t()
    bg, bu = _sum_bound(xv, guv[:F]), _sum_bound(xv, guv[F:])
    act = plain.activation(gate, "silu")
    # silu rises by less than 1.1 times its argument; 2^-18 for its own few instructions
    _check(h, act * up, (1.1 * bg + 2.0 ** -18 * (act.abs() + 2.0 ** -10)) * (up.abs() + bu) + act.abs() * bu, dtype)
    hv = plain.rounded(h) if quantized else h.double()
    exact = hv @ dv.t()
    _check(out, exact + res.double(), _sum_bound(hv, dv) + 2.0 ** -23 * exact.abs(), torch.float32)
    for _ in range(20):
        again = res.clone()
        _feed_forward(m, x, gate_up, down, quantized, again)
        assert torch.equal(again, out)


def test_other_streams():
    """Two streams at once, products that split K over clusters on both and few tokens, many and 4-bit ones between them: as one after the other."""
    m = mx()
    w, _ = _matrix(1200, 8192, 1, 4.0)
    v, _ = _matrix(700, 4096, 2, 4.0)
    g = torch.Generator().manual_seed(0)
    calls = []
    for tokens in (1, 14, 60, 128, 300):
        for mat in (w, v):
            x = torch.randn(tokens, mat.columns, generator=g).half().to(DEV)
            calls.append((x, mat))
    want = []
    for x, mat in calls:
        for q in (False, True):
            o = torch.empty(x.shape[0], mat.rows, device=DEV)
            m.gemm_mxfp4(m.quantize_mxfp4(x) if q else x, mat, o)
            want.append(o)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(3):
        got = [[], []]
        for i, (x, mat) in enumerate(calls):
            for q in (False, True):
                for s in (0, 1):
                    with torch.cuda.stream(streams[s]):
                        # the second stream walks the list backwards
                        y, mt = (x, mat) if s == 0 else calls[len(calls) - 1 - i]
                        o = torch.empty(y.shape[0], mt.rows, device=DEV)
                        m.gemm_mxfp4(m.quantize_mxfp4(y) if q else y, mt, o)
                        got[s].append(o)
        torch.cuda.synchronize()
    ops().raise_on_device_error()
    n = len(calls)
    for i in range(n):
        for q in (0, 1):
            assert torch.equal(got[0][2 * i + q], want[2 * i + q])
            assert torch.equal(got[1][2 * i + q], want[2 * (n - 1 - i) + q])


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("tokens", [3, 40, 600])
def test_two_captured_graphs(tokens, quantized):
    """Two graphs of the same operators (workspaces and all), replayed in turn, on new inputs, and both at once on two streams."""
    m = mx()
    H, F = 512, 1536
    gate_up, _ = _matrix(2 * F, H, 7, 4.0)
    down, _ = _matrix(H, F, 8, 4.0)
    g = torch.Generator().manual_seed(tokens)
    xs = [torch.zeros(tokens, H, device=DEV, dtype=torch.bfloat16) for _ in range(2)]
    outs = [torch.zeros(tokens, H, device=DEV) for _ in range(2)]
    graphs = []
    for x, out in zip(xs, outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):                     # the first call with these sizes may be one that is captured
            out.zero_()
            _feed_forward(m, x, gate_up, down, quantized, out)
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(3):
        want = []
        for x in xs:
            x.copy_(torch.randn(tokens, H, generator=g))
            out = torch.zeros(tokens, H, device=DEV)
            _feed_forward(m, x, gate_up, down, quantized, out)
            want.append(out)
        torch.cuda.synchronize()
        if turn < 2:
            for graph in graphs:
                graph.replay()
        else:
            for graph, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        ops().raise_on_device_error()
        for out, want_one in zip(outs, want):
            assert torch.equal(out, want_one)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens", [1, 5, 16, 40, 200])
def test_infinities_and_nans_of_activations(tokens, dtype):
    m = mx()
    K = 640
    w, wv = _matrix(96, K, tokens)
    a = torch.randn(tokens, K, generator=torch.Generator().manual_seed(tokens)).to(dtype).to(DEV)
    a[0, 3] = float("inf")
    if tokens > 1:
        a[1, 600] = float("-inf")
        a[tokens - 1, 100] = float("nan")
    if tokens > 4:
        a[2, 5], a[2, 300] = float("inf"), float("-inf")
    out = torch.zeros(tokens, 96, device=DEV)
    m.gemm_mxfp4(a, w, out)
    ops().raise_on_device_error()
    # term by term: a sum is NaN with a NaN term (an infinity times zero is one) or infinities of both signs, infinite with one of either
    terms = a.double().unsqueeze(1) * wv.unsqueeze(0)
    plus, minus = (terms == float("inf")).any(-1), (terms == -float("inf")).any(-1)
    nan = terms.isnan().any(-1) | (plus & minus)
    assert torch.equal(out.isnan(), nan)
    assert torch.equal((out == float("inf")) & ~nan, plus & ~nan) and torch.equal((out == -float("inf")) & ~nan, minus & ~nan)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens", [4, 40, 300])
def test_rows_that_are_one_row(tokens, dtype):
    """Activations that are one row told over and over (pitch 0) or overlap; a single row whose pitch says nothing; both operands the same matrix."""
    m = mx()
    K = 256
    w, wv = _matrix(136, K, tokens)
    row = torch.randn(K + 8 * tokens, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    for a in (row[:K].unsqueeze(0).expand(tokens, K), row.as_strided((tokens, K), (8, 1)), row.as_strided((1, K), (3, 1)), row.as_strided((1, K), (0, 1))):
        out = torch.empty(a.shape[0], 136, device=DEV, dtype=dtype)
        m.gemm_mxfp4(a, w, out)
        ops().raise_on_device_error()
        _check(out, a.double() @ wv.t(), _sum_bound(a.double(), wv), dtype)
        q = m.quantize_mxfp4(a)
        assert torch.equal(m.dequantize_mxfp4(q, torch.float32).double(), plain.rounded(a))
    out = torch.empty(136, 136, device=DEV)
    m.gemm_mxfp4(w, w, out)
    _check(out, wv @ wv.t(), _sum_bound(wv, wv), torch.float32)


def test_results_whose_rows_overlap_are_refused():
    m = mx()
    w, _ = _matrix(64, 96, 1)
    a, flat = torch.zeros(4, 96, device=DEV), torch.zeros(400, device=DEV)
    for out in (flat[:64].unsqueeze(0).expand(4, 64), flat.as_strided((4, 64), (60, 1))):
        with pytest.raises(m.KernelError, match="overlap"):
            m.gemm_mxfp4(a, w, out)
    with pytest.raises(m.KernelError, match="overlap"):
        m.dequantize_mxfp4(w, out=flat.as_strided((64, 96), (4, 1)))
    assert bool((flat == 0).all())


def test_codes_beyond_4_gigabytes():
    """A matrix of 140,001 rows by 65,568 columns, 4.6 GB of codes: its last rows count like the first."""
    m = mx()
    N, K = 140001, 65568
    blocks = K // 32
    g = torch.Generator(device=DEV).manual_seed(3)
    codes = torch.empty(N, blocks * 16, device=DEV, dtype=torch.uint8)
    codes.random_(0, 256, generator=g)
    scales = torch.empty(N, blocks, device=DEV, dtype=torch.uint8)
    scales.random_(118, 126, generator=g)
    w = m.Mxfp4Matrix(codes, scales)
    rows = torch.tensor([0, 1, 65535, 65536, 65537, 131072, 139999, N - 1], device=DEV)
    part = m.Mxfp4Matrix(codes[rows].contiguous(), scales[rows].contiguous())
    wv = m.dequantize_mxfp4(part, torch.float32).double()
    for tokens, dtype, quantized in ((1, torch.bfloat16, False), (3, torch.float32, False), (20, torch.float16, False), (20, torch.bfloat16, True),
                                     (150, torch.bfloat16, False), (150, torch.bfloat16, True)):
        a = torch.randn(tokens, K, device=DEV, generator=g).to(dtype)
        out = torch.empty(tokens, N, device=DEV, dtype=torch.float32 if dtype is torch.float32 else dtype)
        q = m.quantize_mxfp4(a)
        m.gemm_mxfp4(q if quantized else a, w, out)
        ops().raise_on_device_error()
        av = m.dequantize_mxfp4(q, torch.float32).double() if quantized else a.double()
        _check(out[:, rows], av @ wv.t(), _sum_bound(av, wv), out.dtype)


def test_values_beyond_4_gigabytes():
    """More than 2^31 values to 4 bits and back, and a result of as many."""
    m = mx()
    rows, K = 70001, 32768
    x = torch.empty(rows, K, device=DEV, dtype=torch.bfloat16)
    x.normal_(generator=torch.Generator(device=DEV).manual_seed(4))
    q = m.quantize_mxfp4(x)
    y = m.dequantize_mxfp4(q)
    for at in (0, 65535, 65536, rows - 2):
        assert torch.equal(y[at:at + 2].double(), plain.rounded(x[at:at + 2]))
    del x, y, q
    torch.cuda.empty_cache()
    w, wv = _matrix(40000, 32, 9)
    a = torch.randn(70001, 32, generator=torch.Generator().manual_seed(5)).bfloat16().to(DEV)
    for operand, av in ((a, a.double()), (m.quantize_mxfp4(a), plain.rounded(a))):
        out = torch.empty(70001, 40000, device=DEV, dtype=torch.bfloat16)
        m.gemm_mxfp4(operand, w, out)
        ops().raise_on_device_error()
        for at in (0, 53687, 65535, 69990):
            _check(out[at:at + 11], av[at:at + 11] @ wv.t(), _sum_bound(av[at:at + 11], wv), torch.bfloat16)
        del out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", [(1040, 6000, 288), (700, 20000, 160), (1500, 9001, 544)])
def test_tiles_of_an_odd_number_of_stages(M, N, K, dtype):
    """Blocks that walk over several tiles whose stages fill their places unevenly: the first result is right, all others are the same."""
    m = mx()
    w, wv = _matrix(N, K, 11)
    a = torch.randn(M, K, generator=torch.Generator().manual_seed(K)).to(dtype).to(DEV)
    first = torch.empty(M, N, device=DEV, dtype=dtype)
    m.gemm_mxfp4(a, w, first)
    _check(first, a.double() @ wv.t(), _sum_bound(a.double(), wv), dtype)
    out = torch.empty_like(first)
    for i in range(40):
        if i % 4 == 0:
            out.fill_(float("nan"))                       # a kernel between them: blocks begin at other times
        m.gemm_mxfp4(a, w, out)
        assert torch.equal(out, first)
    ops().raise_on_device_error()
