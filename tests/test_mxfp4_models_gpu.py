"""4-bit matrices in every architecture: each product that a model's steps make is held to its definition in 64 bits on the very inputs it got (logits of two
whole runs would differ by what random models make of roundings)."""
import pytest
import torch

from plain import mxfp4_plain as plain
from test_mxfp4_gpu import DEV, _check, _sum_bound, mx, ops

pytestmark = pytest.mark.gpu


def _model(which):
    from pifelix_helpers import CONFIGS as P, PifelixModel
    from resatar_helpers import CONFIGS as R, ResatarModel
    from taborax_helpers import CONFIGS as T, TaboraxModel
    from tutelix_helpers import CONFIGS as U, TutelixModel
    from vononex_helpers import CONFIGS as V, VononexModel
    from vozirax_helpers import CONFIGS as Z, VoziraxModel
    kind, letter = which.split("-")
    configs, cls = {"Pifelix": (P, PifelixModel), "Resatar": (R, ResatarModel), "Taborax": (T, TaboraxModel), "Tutelix": (U, TutelixModel),
                    "Vononex": (V, VononexModel), "Vozirax": (Z, VoziraxModel)}[kind]
    return cls(configs[letter], seed=7)


def _engine(folder, amp, activations, n_positions=256):
    from transformers_neuronx_b200 import NeuronAutoModelForCausalLM, NeuronConfig, QuantizationConfig
    model = NeuronAutoModelForCausalLM.from_pretrained(folder, batch_size=2, amp=amp, n_positions=n_positions, neuron_config=NeuronConfig(
        quant=QuantizationConfig(activation_quant_dtype=activations), output_all_logits=True))
    return model.to_neuron()


def _steps(model, ids, steps):
    """A prompt's logits and those of `steps` single tokens behind it."""
    out = [model.forward(torch.tensor(ids))]
    for t in range(steps):
        out.append(model.forward(torch.full((len(ids), 1), 7 + t, dtype=torch.long), torch.tensor([len(ids[0]) + t])))
    return out


def _values(m, x):
    return plain.values(plain.unpack(x.codes), x.scales, x.columns) if isinstance(x, m.Mxfp4Matrix) else x.double()


def _watch(m, monkeypatch):
    """Puts a check behind every product and every quantisation of the module; returns the list of what was checked."""
    seen, gemm, gated, quantize = [], m.gemm_mxfp4, m.gated_gemm_mxfp4, m.quantize_mxfp4

    def sums(a, w, bias):
        av, wv = _values(m, a), _values(m, w)
        s = av @ wv.t() + (bias.double() if bias is not None else 0.0)
        return s, _sum_bound(av, wv) + 2.0 ** -23 * (s.abs() + (bias.double().abs() if bias is not None else 0.0))

    def through(s, off, act):
        """act(s) and how far it may be off: slopes are at most 1.13 (relu2: 2 |x|), 2^-18 of the argument's size for the activation itself."""
        if act in (None, "none"):
            return s, off
        act = {"swish": "silu", "gelu_pytorch_tanh": "gelu_new", "gelu_new_legacy": "gelu_new"}.get(act, act)
        slope = 2 * (s.abs() + off) if act == "relu2" else 1.13
        return plain.activation(s, act), slope * off + 2.0 ** -18 * s.abs()

    def checked_gemm(a, w, out, bias=None, residual=None, activation=None):
        res = residual.double() if residual is not None else None              # before it is written over
        got = gemm(a, w, out, bias=bias, residual=residual, activation=activation)
        want, off = through(*sums(a, w, bias), activation)
        if res is not None:
            want = want + res
        _check(got, want, off, out.dtype)
        seen.append(("gemm", isinstance(a, m.Mxfp4Matrix), want.shape))
        return got

    def checked_gated(a, w, out, bias=None, activation="silu"):
        got = gated(a, w, out, bias=bias, activation=activation)
        s, off = sums(a, w, bias)
        F = s.shape[1] // 2
        gate, off_gate = through(s[:, :F], off[:, :F], activation)
        up, off_up = s[:, F:], off[:, F:]
        _check(got, gate * up, off_gate * up.abs() + gate.abs() * off_up + off_gate * off_up + 2.0 ** -23 * (gate * up).abs(), out.dtype)
        seen.append(("gated", isinstance(a, m.Mxfp4Matrix), gate.shape))
        return got

    def checked_quantize(x, out=None):
        got = quantize(x, out)
        code, scale = plain.quantize(x)
        assert torch.equal(got.codes, plain.pack(code)) and torch.equal(got.scales, scale)
        seen.append(("quantize", True, x.shape))
        return got

    monkeypatch.setattr(m, "gemm_mxfp4", checked_gemm)
    monkeypatch.setattr(m, "gated_gemm_mxfp4", checked_gated)
    monkeypatch.setattr(m, "quantize_mxfp4", checked_quantize)
    return seen


@pytest.mark.parametrize("activations", [None, "mxfp4"])
@pytest.mark.parametrize("amp", ["bf16", "f16"])
@pytest.mark.parametrize("which", ["Vononex-Q", "Pifelix-B", "Tutelix-B", "Tutelix-D", "Vozirax-B", "Resatar-B", "Taborax-B", "Taborax-D"])
def test_every_product_of_a_model(which, amp, activations, monkeypatch):
    m, o = mx(), ops()
    tiny = _model(which)
    model = _engine(tiny.folder, amp, activations)
    model.engine.runner.use_cuda_graphs = False
    linears = [l for b in model.model.blocks for p in (b.mixer, b.feed_forward) if p is not None for l in p.linears()]
    assert linears and any(l.quantized for l in linears)
    assert all(l.quantized == (l.weight.shape[1] % 32 == 0) for l in linears)
    scaled, activate = [], o.gated_activation

    def watched(gu, a, activation, row_scale=None):
        if row_scale is not None:
            scaled.append(gu.shape)
        return activate(gu, a, activation, row_scale)
    monkeypatch.setattr(o, "gated_activation", watched)
    seen = _watch(m, monkeypatch)
    logits = _steps(model, [tiny.random_ids(150, seed=s) for s in (1, 2)], 2)
    o.raise_on_device_error()
    assert all(bool(torch.isfinite(x).all()) for x in logits)
    kinds = {(kind, q) for kind, q, _ in seen if kind != "quantize"}
    assert kinds and {q for _, q in kinds} == {activations is not None}
    tokens = {shape[0] for _, _, shape in seen}
    assert max(tokens) > 128 and min(tokens) <= 2              # both ends: a prompt and single tokens
    if which == "Taborax-B":                                   # a shared expert with a gate of its own, whose width the routed ones do not divide
        assert scaled and any(kind == "gemm" for kind, _ in kinds)


@pytest.mark.parametrize("amp", ["f16", "bf16"])
@pytest.mark.parametrize("which", ["Vononex-Q", "Tutelix-B", "Vozirax-B", "Resatar-B", "Taborax-B"])
def test_a_model_loads_only_the_libraries_it_names(which, amp, monkeypatch):
    """4-bit inputs, whose type says nothing about the engine's: nothing is left to be compiled within a request."""
    from transformers_neuronx_b200.kernels import build
    m = mx()
    tiny = _model(which)
    model = _engine(tiny.folder, amp, "mxfp4")
    named = set(build.with_flavour(model.model.libraries(model.model.act_dtype), model.model.act_dtype))
    asked, load = set(), build.load

    def recording(name, dtype=None):
        if "mxfp4" in name:
            f = build.flavour_of(dtype)
            asked.add(f"{name}.{f}" if f else name)
        return load(name, dtype)
    monkeypatch.setattr(build, "load", recording)
    monkeypatch.setattr(m, "_entries", {})
    monkeypatch.setattr(m, "_tiles", {})
    _steps(model, [tiny.random_ids(150, seed=s) for s in (1, 2)], 1)
    assert asked and asked <= named, sorted(asked - named)


@pytest.mark.parametrize("amp", ["f16", "bf16", "f32"])
def test_a_saved_model_keeps_the_builds_it_runs(amp, tmp_path):
    """save() writes the libraries of the engine's own type, those of its 4-bit matrices among them."""
    import os
    from helpers import TinyModel
    from transformers_neuronx_b200 import NeuronConfig, QuantizationConfig
    from transformers_neuronx_b200.kernels import build
    from transformers_neuronx_b200.opt.model import OPTForSampling
    tiny = TinyModel("A", seed=1)
    model = OPTForSampling.from_pretrained(tiny.folder, batch_size=1, amp=amp, n_positions=32,
                                           neuron_config=NeuronConfig(quant=None if amp == "f32" else QuantizationConfig(activation_quant_dtype="mxfp4")))
    model.to_neuron()
    model.save(str(tmp_path))
    act = model.model.act_dtype
    named = build.with_flavour(model.model.libraries(act), act)
    assert amp == "f32" or build.with_flavour(["gemm_mxfp4_tiles"], act)[0] in named
    assert sorted(os.listdir(tmp_path)) == sorted(os.path.basename(build.library_path(n)) for n in named)
