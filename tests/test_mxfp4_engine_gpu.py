"""4-bit matrices through the engine's own entry points: a model whose projections were quantized against the same model with the 16-bit
values that the 4 bits stand for; captured steps against eager ones; choices of what is quantized."""
import warnings

import pytest
import torch

from helpers import TOLERANCE, TinyModel, rel_error
from plain import mxfp4_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"bf16": ("bfloat16", torch.bfloat16), "f16": ("float16", torch.float16)}
WIDE = dict(hidden_size=256, ffn_dim=512, word_embed_proj_dim=256, num_attention_heads=4, max_position_embeddings=400)


def _opt(folder, amp, quant, n_positions=320, batch=2):
    from transformers_neuronx_b200 import NeuronConfig
    from transformers_neuronx_b200.opt.model import OPTForSampling
    model = OPTForSampling.from_pretrained(folder, batch_size=batch, amp=amp, n_positions=n_positions,
                                           neuron_config=NeuronConfig(quant=quant, output_all_logits=True))
    model.to_neuron()
    return model


def _linears(model):
    return [l for b in model.model.blocks for p in (b.mixer, b.feed_forward) if p is not None for l in p.linears()]


def _as_16_bits(model):
    """The matrices that quantization would bring into 4 bits, as 16-bit matrices of the values that they then stand for."""
    from transformers_neuronx_b200.kernels import mxfp4
    for l in _linears(model):
        if l.weight.shape[1] % 32 == 0:
            l.weight = mxfp4.dequantize_mxfp4(mxfp4.quantize_mxfp4(l.weight), l.weight.dtype)


def _run(model, ids, steps):
    """Logits of a prompt and of `steps` decode steps behind it."""
    out = [model.forward(torch.tensor(ids))]
    n = len(ids[0])
    for t in range(steps):
        out.append(model.forward(torch.full((len(ids), 1), 7 + t, dtype=torch.long), torch.tensor([n + t])))
    return [o.float().cpu() for o in out]


@pytest.mark.parametrize("amp", ["bf16", "f16"])
@pytest.mark.parametrize("length", [5, 40, 300])
def test_opt_against_its_own_values(amp, length):
    """One token to more than a tile of the prompts' kernel, then single tokens."""
    from transformers_neuronx_b200 import QuantizationConfig
    from transformers_neuronx_b200.kernels import ops
    tiny = TinyModel("A", seed=11, matrix_dtype=TYPES[amp][1], overrides=WIDE)
    ids = [tiny.random_ids(length, seed=s) for s in (1, 2)]
    quantized, same = _opt(tiny.folder, amp, QuantizationConfig()), _opt(tiny.folder, amp, None)
    _as_16_bits(same)
    assert all(l.quantized for l in _linears(quantized)) and not any(l.quantized for l in _linears(same))
    before = sum(l.weight.numel() * 2 for l in _linears(same))
    assert sum(l.weight.nbytes() for l in _linears(quantized)) * 64 == before * 17        # 17 bytes for 32 values
    for got, want in zip(_run(quantized, ids, 4), _run(same, ids, 4)):
        assert rel_error(got, want) <= TOLERANCE[TYPES[amp][0]]
    ops.raise_on_device_error()


def test_vononex_against_its_own_values():
    """Gated feed-forwards (their front half is one kernel), parallel mixers' joined projections, recurrent mixers."""
    from vononex_helpers import CONFIGS, BF16_NINTH_DECILE, BF16_WORST, TOLERANCE as TOL, VononexModel
    from transformers_neuronx_b200 import NeuronAutoModelForCausalLM, NeuronConfig, QuantizationConfig
    from transformers_neuronx_b200.kernels import ops
    from transformers_neuronx_b200.parts.feedforward import GatedDenseFeedForward
    tiny = VononexModel(CONFIGS["Q"], seed=5)
    ids = [tiny.random_ids(150, seed=s) for s in (1, 2)]
    logits = []
    for quant in (QuantizationConfig(), None):
        model = NeuronAutoModelForCausalLM.from_pretrained(tiny.folder, batch_size=2, amp="bf16", n_positions=256,
                                                           neuron_config=NeuronConfig(quant=quant, output_all_logits=True))
        model.to_neuron()
        if quant is None:
            _as_16_bits(model)
        else:
            assert any(isinstance(b.feed_forward, GatedDenseFeedForward) and b.feed_forward.gate_up.quantized for b in model.model.blocks)
        logits.append(_run(model, ids, 3))
    ops.raise_on_device_error()
    for got, want in zip(*logits):
        rows = (got - want).abs().amax(-1) / want.abs().amax(-1)
        rows = rows.flatten().sort().values
        n = len(rows)
        assert float(rows[n // 2]) <= TOL["bfloat16"] and float(rows[int(0.9 * (n - 1))]) <= BF16_NINTH_DECILE and float(rows[-1]) <= BF16_WORST


@pytest.mark.parametrize("activations", [None, "mxfp4"])
def test_captured_steps(activations):
    """Steps replayed as graphs leave what eager ones leave: the same kernels on the same inputs."""
    from transformers_neuronx_b200 import QuantizationConfig
    tiny = TinyModel("A", seed=12, overrides=WIDE)
    ids = [tiny.random_ids(20, seed=s) for s in (1, 2)]
    quant = QuantizationConfig(activation_quant_dtype=activations)
    graphs, eager = _opt(tiny.folder, "bf16", quant), _opt(tiny.folder, "bf16", quant)
    eager.engine.runner.use_cuda_graphs = False
    for got, want in zip(_run(graphs, ids, 8), _run(eager, ids, 8)):
        assert torch.equal(got, want) and bool(torch.isfinite(got).all())
    graphs.reset()
    eager.reset()
    out = graphs.sample(torch.tensor(ids), sequence_length=40, top_k=1)
    assert torch.equal(out, eager.sample(torch.tensor(ids), sequence_length=40, top_k=1))


def test_linear_with_4_bit_activations():
    """A projection rounds its input, then multiplies: against both steps in 64 bits."""
    from transformers_neuronx_b200 import QuantizationConfig
    tiny = TinyModel("A", seed=13, overrides=WIDE)
    model = _opt(tiny.folder, "bf16", QuantizationConfig(activation_quant_dtype="mxfp4"))
    fc2 = model.model.blocks[0].feed_forward.fc2
    for tokens in (1, 33, 200):
        a = torch.randn(tokens, 512, generator=torch.Generator().manual_seed(tokens)).bfloat16().to(DEV)
        res = torch.randn(tokens, 256, generator=torch.Generator().manual_seed(tokens)).to(DEV)
        w = plain.values(plain.unpack(fc2.weight.codes), fc2.weight.scales, 512)
        av = plain.rounded(a)
        want = av @ w.t() + fc2.bias.double() + res.double()
        out = res.clone()
        fc2.forward(a, out, residual=out)
        bound = (32 * 2.0 ** -22 + 64 * 2.0 ** -24) * (av.abs() @ w.abs().t()) + 2.0 ** -22 * (want.abs() + fc2.bias.double().abs() + res.double().abs())
        assert bool(((out.double() - want).abs() <= bound).all())


def test_what_is_quantized():
    from transformers_neuronx_b200 import QuantizationConfig
    tiny = TinyModel("A", seed=14, overrides=dict(WIDE, ffn_dim=520))                       # 520 columns are no whole blocks
    model = _opt(tiny.folder, "bf16", QuantizationConfig())
    ff, mixer = model.model.blocks[0].feed_forward, model.model.blocks[0].mixer
    assert ff.fc1.quantized and not ff.fc2.quantized and mixer.qkv.quantized and mixer.out.quantized
    model = _opt(tiny.folder, "bf16", QuantizationConfig(quantize_attn=False))
    assert model.model.blocks[1].feed_forward.fc1.quantized and not model.model.blocks[1].mixer.qkv.quantized
    model = _opt(tiny.folder, "bf16", QuantizationConfig(no_quantize_list=["layers.1.self_attn.k_proj", "fc1"]))
    assert model.model.blocks[0].mixer.qkv.quantized and not model.model.blocks[1].mixer.qkv.quantized      # joined with it
    assert not model.model.blocks[0].feed_forward.fc1.quantized
    assert torch.isfinite(model.forward(torch.tensor([tiny.random_ids(9, seed=1)] * 2))).all()
    with pytest.raises(ValueError):
        _opt(tiny.folder, "f32", QuantizationConfig())
    stored_32 = TinyModel("A", seed=14, matrix_dtype=torch.float32, overrides=WIDE)          # 32-bit matrices stay
    with warnings.catch_warnings(record=True) as w:
        warnings.simplefilter("always")
        model = _opt(stored_32.folder, "bf16", QuantizationConfig())
    assert any("4 bits" in str(x.message) for x in w) and not any(l.quantized for l in _linears(model))


def test_demo_and_profile(tmp_path, capsys):
    from transformers_neuronx_b200.opt.demo import main
    tiny = TinyModel("A", seed=15, overrides=WIDE)
    main(["--amp", "bf16", "run", tiny.folder, "--batch_size", "2", "--n_positions", "24", "--weight_format", "mxfp4", "--activation_format", "mxfp4"])
    assert "generated_sequence=" in capsys.readouterr().out
    from transformers_neuronx_b200 import QuantizationConfig
    model = _opt(tiny.folder, "f16", QuantizationConfig(activation_quant_dtype="mxfp4"))
    report = model.profile(str(tmp_path))
    assert "gemm_mxfp4" in report and "quantize_mxfp4" in report
    assert model.is_compiled()
