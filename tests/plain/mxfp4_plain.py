"""Microscaled 4-bit numbers in 64 bits on the CPU or the GPU: the definition, value by value."""
import torch

MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def quantize(x):
    """x [rows, K] -> (codes uint8 [rows, blocks, 32], scale bytes uint8 [rows, blocks])."""
    x = x.double()
    rows, k = x.shape
    x = torch.cat((x, x.new_zeros(rows, -k % 32)), 1).view(rows, -1, 32)
    bad = ~torch.isfinite(x).all(-1)
    m = torch.where(bad.unsqueeze(-1), torch.zeros_like(x), x).abs().amax(-1)
    e = torch.full_like(m, -127.0)
    for n in range(-126, 128):                              # the smallest exponent that cuts nothing off, found by trying them all
        e = torch.where(m > 6 * 2.0 ** (n - 1), torch.full_like(e, float(n)), e)
    v = x / torch.exp2(e).unsqueeze(-1)
    mags = torch.tensor(MAGNITUDES, dtype=torch.float64, device=x.device)
    d = (v.abs().unsqueeze(-1) - mags).abs()
    d = torch.where(d.isnan(), torch.zeros_like(d), d)
    near = d.amin(-1, keepdim=True) == d                    # one code, or two that are as near: the even one of them
    code = torch.where(near, torch.arange(8, device=x.device) + 100 * (torch.arange(8, device=x.device) % 2), torch.tensor(1000, device=x.device)).amin(-1) % 100
    code = code + 8 * torch.signbit(x).long()
    scale = (e + 127).long()
    code = torch.where(bad.unsqueeze(-1), torch.zeros_like(code), code)
    scale = torch.where(bad, torch.full_like(scale, 255), scale)
    return code.to(torch.uint8), scale.to(torch.uint8)


def pack(code):
    """Codes [rows, blocks, 32] -> bytes [rows, blocks * 16], value 2j in the low half of byte j."""
    c = code.flatten(1)
    return (c[:, 0::2] | (c[:, 1::2] << 4)).contiguous()


def unpack(codes):
    return torch.stack((codes & 15, codes >> 4), -1).flatten(1).view(codes.shape[0], -1, 32)


def values(code, scale, k):
    """Codes [rows, blocks, 32] and scale bytes -> 64-bit values [rows, k]."""
    mags = torch.tensor(MAGNITUDES, dtype=torch.float64, device=code.device)
    v = mags[(code & 7).long()] * (1.0 - 2.0 * (code >> 3).double())
    s = torch.exp2(scale.double() - 127)
    s = torch.where(scale == 255, torch.full_like(s, float("nan")), s)
    return (v * s.unsqueeze(-1)).flatten(1)[:, :k]


def rounded(x):
    """x as it stands in 4 bits, in 64 bits."""
    return values(*quantize(x), x.shape[1])


def activation(x, name):
    if name in (None, "none"):
        return x
    if name == "relu":
        return x.clamp_min(0)
    if name == "relu2":
        return x.clamp_min(0) ** 2
    if name == "silu":
        return x * torch.sigmoid(x)
    if name == "sigmoid":
        return torch.sigmoid(x)
    if name == "gelu":
        return 0.5 * x * (1 + torch.erf(x * 0.7071067811865476))
    assert name == "gelu_new"
    return 0.5 * x * (1 + torch.tanh(0.7978845608028654 * (x + 0.044715 * x ** 3)))
