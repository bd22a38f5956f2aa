"""4-bit matrices without a GPU: the type's checks, the plain form that the GPU tests compare with."""
import pytest
import torch

from plain import mxfp4_plain as plain


def mx():
    from transformers_neuronx_b200.kernels import mxfp4
    return mxfp4


def test_matrix_refusals():
    m = mx()
    codes, scales = torch.zeros(5, 48, dtype=torch.uint8), torch.zeros(5, 3, dtype=torch.uint8)
    assert m.Mxfp4Matrix(codes, scales).shape == (5, 96)
    assert m.Mxfp4Matrix(codes, scales, 65).shape == (5, 65) and m.Mxfp4Matrix(codes, scales, 65).numel() == 325
    for bad in ((codes.int(), scales, None), (codes, scales.int(), None), (codes[:4], scales, None), (codes[:, :32], scales, None),
                (codes, scales, 64), (codes, scales, 97), (codes, scales, 0), (codes.t(), scales, None), (codes, scales[0], None),
                (codes[:, :0], scales[:, :0], None), (torch.zeros(5, 96, dtype=torch.uint8)[:, :48], scales, None), (None, scales, None)):
        with pytest.raises(m.KernelError):
            m.Mxfp4Matrix(*bad)


def test_refused_off_the_gpu():
    m = mx()
    w = m.Mxfp4Matrix(torch.zeros(5, 48, dtype=torch.uint8), torch.zeros(5, 3, dtype=torch.uint8))
    x, out = torch.zeros(2, 96), torch.zeros(2, 5)
    for call in (lambda: m.quantize_mxfp4(x), lambda: m.dequantize_mxfp4(w), lambda: m.gemm_mxfp4(x, w, out),
                 lambda: m.gated_gemm_mxfp4(x, w, out), lambda: m.gemm_mxfp4(x, x, out)):
        with pytest.raises(m.KernelError):
            call()


def test_plain_rounding():
    """The plain form itself, on values that can be checked by eye: ties, the scale's border, signed zeros, what is not finite."""
    x = torch.zeros(1, 64)
    x[0, :14] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -0.0, 0.26, 5.01, -3.49, 1e-9])
    code, scale = plain.quantize(x)
    assert scale.tolist() == [[127, 0]]
    assert code[0, 0, :14].tolist() == [7, 0, 2, 2, 4, 4, 6, 6, 8, 8, 1, 7, 13, 0]
    y = torch.zeros(1, 32); y[0, 0] = 6.0001
    assert plain.quantize(y)[1].tolist() == [[128]]
    y[0, 1] = float("inf")
    assert plain.quantize(y)[1].tolist() == [[255]] and plain.rounded(y).isnan().all()
    assert torch.equal(plain.unpack(plain.pack(code)), code)
    tiny = torch.full((1, 32), 2.0 ** -140)
    assert plain.quantize(tiny)[1].tolist() == [[0]] and float(plain.rounded(tiny).abs().max()) == 0.0


def test_quantization_config():
    from transformers_neuronx_b200 import NeuronConfig, QuantizationConfig
    q = QuantizationConfig(no_quantize_list=["fc2"])
    assert (q.quant_dtype, q.activation_quant_dtype, q.quantize_attn, q.no_quantize_list) == ("mxfp4", None, True, ["fc2"])
    assert NeuronConfig(quant=q).quant is q and NeuronConfig(quant=q).ignored == {} and NeuronConfig().quant is None
    for bad, error in ((dict(quant_dtype="s8"), NotImplementedError), (dict(activation_quant_dtype="s8"), NotImplementedError),
                       (dict(no_quantize_list="fc2"), TypeError)):
        with pytest.raises(error):
            QuantizationConfig(**bad)


def test_quantized_models_need_16_bits():
    from helpers import TinyModel
    from transformers_neuronx_b200 import QuantizationConfig
    from transformers_neuronx_b200.models import opt as opt_arch
    from transformers_neuronx_b200.models.decoder import DecoderModel
    tiny = TinyModel("A", seed=1)
    model = DecoderModel(opt_arch.build_spec(tiny.cfg))
    assert "gemv_mxfp4" not in model.libraries(torch.bfloat16)
    model.act_dtype = torch.float32
    with pytest.raises(ValueError):
        model.quantize(QuantizationConfig())
    model.quantization = QuantizationConfig()
    assert {"mxfp4", "gemv_mxfp4", "gemm_mxfp4", "gemm_mxfp4_tiles"} <= set(model.libraries(torch.bfloat16))


def test_sizes_that_kernels_do_not_count_are_refused():
    """Rows and columns are counted in 32 bits: larger ones are refused before anything runs."""
    m = mx()
    with pytest.raises(m.KernelError, match="at most"):
        m.Mxfp4Matrix(torch.empty(2 ** 31, 16, dtype=torch.uint8, device="meta"), torch.empty(2 ** 31, 1, dtype=torch.uint8, device="meta"))
    x = torch.empty(1, 32).expand(2 ** 31, 32)
    with pytest.raises(m.KernelError, match="at most"):
        m._floats(x, "x", x.get_device())
    one = torch.empty_strided((1, 20), (3, 1))
    assert m._floats(one, "x", one.get_device()) == (1, 20, 24)            # the pitch of one row means nothing
