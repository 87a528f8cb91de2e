"""The layers that run the sequence and normalisation operators together."""

import pytest
import torch

import trnfft_b200 as trnfft
from trnfft_b200 import ComplexTensor
from trnfft_b200.nn import ComplexDecayAttention, ComplexGroupNorm
from tests.layer_refs import decay_ref, norm_ref

pytestmark = pytest.mark.gpu


def cplx(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return ComplexTensor(torch.randn(*shape, device="cuda", generator=g), torch.randn(*shape, device="cuda", generator=g))


def layer_ref(m, re, im, state=None):
    """The layer in 64 bits on (batch, frames, features) planes."""
    def linear(p, re, im):
        wr, wi = p.W_re.weight.double(), p.W_im.weight.double()
        yr, yi = re @ wr.T - im @ wi.T, re @ wi.T + im @ wr.T
        return (yr, yi) if p.bias_re is None else (yr + p.bias_re.double(), yi + p.bias_im.double())

    h, w = m.heads, m.head_width
    q, k, v = (torch.cat([x.unflatten(-1, (h, w)) for x in linear(p, re, im)], -1) for p in (m.q, m.k, m.v))
    o, last = decay_ref(q, k, v, m.log_decay, (2 * w) ** -0.5, state)
    b, t = o.shape[:2]
    o = norm_ref(o.reshape(b * t, -1), h, m.norm.weight.double(), m.norm.bias.double(), m.norm.eps, None).view(b, t, h, 2, w)
    yr, yi = linear(m.out, o[..., 0, :].flatten(-2), o[..., 1, :].flatten(-2))
    return yr, yi, last


def test_layer_forward_gradients_and_stream():
    torch.manual_seed(0)
    m = ComplexDecayAttention(12, 3, 8).cuda()
    x = cplx(2, 90, 12)
    y, last = m(x, return_state=True)
    yr, yi, wl = layer_ref(m, x.real.double(), x.imag.double())
    for a, b in ((y.real, yr), (y.imag, yi), (last, wl)):
        assert float((a.double() - b).norm() / b.norm()) < 2e-5
    gr, gi = torch.randn_like(y.real), torch.randn_like(y.imag)
    names, params = zip(*m.named_parameters())
    got = torch.autograd.grad((y.real, y.imag), params, (gr, gi))
    want = torch.autograd.grad((yr, yi), params, (gr.double(), gi.double()))
    for n, a, b in zip(names, got, want):
        assert float((a - b).norm() / b.norm()) < 1e-3, n
    # frame by frame, from an empty state and from the middle
    state = m.initial_state(2)
    for t in range(90):
        f = m.step(x[:, t], state)
        for a, b in ((f.real, yr[:, t]), (f.imag, yi[:, t])):
            assert float((a.double() - b).norm() / b.norm()) < 2e-5
    _, half = m(x[:, :50], return_state=True)
    rest = m(x[:, 50:], state=half)
    assert float((rest.real.double() - yr[:, 50:]).norm() / yr[:, 50:].norm()) < 2e-5


def test_spectrogram_to_spectrogram():
    """STFT, norm of each frame, mixing along time, inverse STFT: a training step and its state."""
    torch.manual_seed(1)
    bins = 33
    norm, mix = ComplexGroupNorm(3, bins).cuda(), ComplexDecayAttention(bins, 2, 16).cuda()
    wave = torch.randn(2, 2000, device="cuda")
    spec = trnfft.stft(wave, n_fft=64, hop_length=16)
    frames = spec.transpose(1, 2)
    h = norm(frames)
    for got, plane, gn in ((h.real, frames.real, norm.gn_re), (h.imag, frames.imag, norm.gn_im)):
        want = norm_ref(plane.double(), 3, gn.weight.double(), gn.bias.double(), gn.eps, None)
        assert float((got.double() - want).norm() / want.norm()) < 1e-5
    out = mix(h)
    y = trnfft.istft(ComplexTensor(out.real, out.imag).transpose(1, 2), n_fft=64, hop_length=16, length=2000)
    assert y.shape == wave.shape
    loss = (out.real ** 2 + out.imag ** 2).sum()
    grads = torch.autograd.grad(loss, [*norm.parameters(), *mix.parameters()])
    assert all(bool(torch.isfinite(g).all()) and float(g.abs().max()) > 0 for g in grads)
