"""Complex-valued layers (same classes as trnfft/nn.py).

``ComplexLinear`` is on the hot path: its forward runs the library's complex
GEMM (``trnfft_b200.nki.dispatch.complex_linear``).  ``ComplexConv1d``,
``ComplexBatchNorm1d`` and ``ComplexModReLU`` are kept for API compatibility
(same parameters and values as trnfft/nn.py:52-129); they are off the FFT hot
path and written as plain torch compositions.  ``GroupNorm``,
``ComplexGroupNorm`` and ``ComplexDecayAttention`` have no counterpart there;
they run the library's group norm and decayed linear attention kernels.
"""

from __future__ import annotations

import math

import torch
import torch.nn as nn

from ._attention import decay_attention, decay_attention_step
from ._norm import group_norm
from .complex import ComplexTensor


class ComplexLinear(nn.Module):
    """Complex-valued linear layer y = W x + b (trnfft/nn.py:18-49).

    Parameters are ``W_re``/``W_im`` (``nn.Linear`` without bias, weight
    shape (out, in)) and ``bias_re``/``bias_im``, initialised like the
    reference (kaiming_uniform with a = sqrt(5), i.e. U(+-1/sqrt(in))).
    """

    def __init__(self, in_features: int, out_features: int, bias: bool = True):
        super().__init__()
        self.W_re = nn.Linear(in_features, out_features, bias=False)
        self.W_im = nn.Linear(in_features, out_features, bias=False)
        self.bias_re = nn.Parameter(torch.zeros(out_features)) if bias else None
        self.bias_im = nn.Parameter(torch.zeros(out_features)) if bias else None
        self._reset_parameters()

    def _reset_parameters(self):
        nn.init.kaiming_uniform_(self.W_re.weight, a=math.sqrt(5))
        nn.init.kaiming_uniform_(self.W_im.weight, a=math.sqrt(5))

    def forward(self, x: ComplexTensor) -> ComplexTensor:
        from . import _gemm

        # the weight's TF32 hi/lo split is cached here and redone only when the
        # weight's storage or version changes (e.g. after an optimizer step)
        if not hasattr(self, "_wsplit"):
            self._wsplit = {}
        if not (self.W_re.weight.is_cuda or x.real.is_cuda):
            self._wsplit = {}
        return _gemm.complex_linear(x, self.W_re.weight, self.W_im.weight, self.bias_re, self.bias_im,
                                    cache=self._wsplit if self.W_re.weight.is_cuda else None)


class ComplexConv1d(nn.Module):
    """Complex 1-D convolution with the reference's parameters (trnfft/nn.py:52-86).

    Parameters: ``conv_re`` / ``conv_im`` (``nn.Conv1d`` without bias, the
    real and imaginary kernel) and optional ``bias_re`` / ``bias_im``.  The
    forward pass runs ONE real convolution over the stacked channels
    [x_re; x_im] with the 2x2 block kernel [[K_re, -K_im], [K_im, K_re]], whose
    output channels are then [y_re; y_im] = [K_re*x_re - K_im*x_im;
    K_im*x_re + K_re*x_im].  Not on the FFT hot path.
    """

    def __init__(self, in_channels: int, out_channels: int, kernel_size: int, stride: int = 1,
                 padding: int = 0, bias: bool = True):
        super().__init__()
        self.conv_re = nn.Conv1d(in_channels, out_channels, kernel_size, stride=stride, padding=padding, bias=False)
        self.conv_im = nn.Conv1d(in_channels, out_channels, kernel_size, stride=stride, padding=padding, bias=False)
        self.bias_re = nn.Parameter(torch.zeros(out_channels)) if bias else None
        self.bias_im = nn.Parameter(torch.zeros(out_channels)) if bias else None

    def forward(self, x: ComplexTensor) -> ComplexTensor:
        kr, ki = self.conv_re.weight, self.conv_im.weight
        block = torch.cat([torch.cat([kr, -ki], dim=1), torch.cat([ki, kr], dim=1)], dim=0)
        b = None
        if self.bias_re is not None:
            b = torch.cat([self.bias_re, self.bias_im])
        y = torch.nn.functional.conv1d(torch.cat([x.real, x.imag], dim=-2), block, b,
                                       stride=self.conv_re.stride, padding=self.conv_re.padding)
        c = kr.shape[0]
        return ComplexTensor(y[..., :c, :], y[..., c:, :])


class ComplexBatchNorm1d(nn.Module):
    """Batch normalisation of the real and the imaginary plane as separate channels
    (trnfft/nn.py:89-104: two independent ``BatchNorm1d``; no whitening of the
    complex covariance).  Keeps the reference's ``bn_re`` / ``bn_im`` modules
    (and state-dict keys); the statistics of each plane are its own."""

    def __init__(self, num_features: int, eps: float = 1e-5):
        super().__init__()
        self.bn_re = nn.BatchNorm1d(num_features, eps=eps)
        self.bn_im = nn.BatchNorm1d(num_features, eps=eps)

    def forward(self, x: ComplexTensor) -> ComplexTensor:
        planes = [bn(p) for bn, p in ((self.bn_re, x.real), (self.bn_im, x.imag))]
        return ComplexTensor(*planes)


class ComplexModReLU(nn.Module):
    """modReLU: keeps the phase of z and maps the modulus r = |z| to max(r + b, 0)
    (trnfft/nn.py:107-129), with one learnt offset b per feature, broadcast
    along the LAST axis as the reference does.  The gain
    max(r + b, 0) / max(r, 1e-8) multiplies both planes."""

    def __init__(self, num_features: int):
        super().__init__()
        self.bias = nn.Parameter(torch.zeros(num_features))

    def forward(self, x: ComplexTensor) -> ComplexTensor:
        r = x.abs()
        gain = torch.relu(r + self.bias) / r.clamp_min(1e-8)
        return ComplexTensor(x.real * gain, x.imag * gain)


class GroupNorm(nn.Module):
    """Group normalisation of channels-last features, with an activation (``trnfft_b200.group_norm``).

    Unlike batch statistics it needs no other sample and no running average, so a stream of
    single frames gets the values that training saw."""

    def __init__(self, num_groups: int, num_channels: int, eps: float = 1e-5, affine: bool = True,
                 activation: str | None = None):
        super().__init__()
        self.num_groups, self.eps, self.activation = num_groups, eps, activation
        self.weight = nn.Parameter(torch.ones(num_channels)) if affine else None
        self.bias = nn.Parameter(torch.zeros(num_channels)) if affine else None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return group_norm(x, self.num_groups, self.weight, self.bias, self.eps, self.activation)


class ComplexGroupNorm(nn.Module):
    """Group normalisation of the real and the imaginary plane, each with its own statistics and
    parameters as in ``ComplexBatchNorm1d``, over channels-last features (batch, ..., channels)."""

    def __init__(self, num_groups: int, num_channels: int, eps: float = 1e-5, activation: str | None = None):
        super().__init__()
        self.gn_re = GroupNorm(num_groups, num_channels, eps, activation=activation)
        self.gn_im = GroupNorm(num_groups, num_channels, eps, activation=activation)

    def forward(self, x: ComplexTensor) -> ComplexTensor:
        return ComplexTensor(self.gn_re(x.real), self.gn_im(x.imag))


class ComplexDecayAttention(nn.Module):
    """Mixing along time for complex features (batch, frames, features): decayed linear attention
    between ``ComplexLinear`` projections, each head's output normalised for itself.

    A head of complex width w (up to 64) is a real head of width 2w over [re, im], so scores are
    Re(q conj(k)).  ``forward`` runs whole sequences; ``step`` one frame (batch, features) of each
    stream on the state that ``forward(..., return_state=True)`` or ``initial_state`` gives, in
    place.  Head h forgets over 2^(3 + 6h/(heads-1)) frames."""

    def __init__(self, features: int, heads: int, head_width: int):
        super().__init__()
        if heads < 1 or not 1 <= head_width <= 64:
            raise ValueError("ComplexDecayAttention: needs a head or more, of a complex width from 1 to 64 (real heads are "
                             f"twice as wide, up to 128), got {heads} of width {head_width}")
        self.heads, self.head_width = heads, head_width
        self.q = ComplexLinear(features, heads * head_width, bias=False)
        self.k = ComplexLinear(features, heads * head_width, bias=False)
        self.v = ComplexLinear(features, heads * head_width, bias=False)
        self.norm = GroupNorm(heads, 2 * heads * head_width)
        self.out = ComplexLinear(heads * head_width, features)
        memory = 2.0 ** (3.0 + 6.0 * torch.arange(heads, dtype=torch.float64) / max(1, heads - 1))
        self.register_buffer("log_decay", torch.log1p(-1.0 / memory).float())

    def _heads(self, x: ComplexTensor) -> torch.Tensor:
        planes = [p.unflatten(-1, (self.heads, self.head_width)) for p in (x.real, x.imag)]
        return torch.cat(planes, dim=-1)

    def _project(self, o: torch.Tensor) -> ComplexTensor:
        o = self.norm(o.reshape(-1, 2 * self.heads * self.head_width)).view(o.shape)
        re, im = (p.flatten(-2) for p in o.split(self.head_width, dim=-1))
        return self.out(ComplexTensor(re, im))

    def initial_state(self, batch: int, device=None) -> torch.Tensor:
        w = 2 * self.head_width
        return torch.zeros(batch, self.heads, w, w, dtype=torch.float32,
                           device=self.log_decay.device if device is None else device)

    def forward(self, x: ComplexTensor, state: torch.Tensor | None = None, return_state: bool = False):
        q, k, v = (self._heads(p(x)) for p in (self.q, self.k, self.v))
        o, last = decay_attention(q, k, v, self.log_decay, initial_state=state, return_state=True)
        y = self._project(o)
        return (y, last) if return_state else y

    @torch.no_grad()
    def step(self, x: ComplexTensor, state: torch.Tensor) -> ComplexTensor:
        q, k, v = (self._heads(p(x)) for p in (self.q, self.k, self.v))
        o, _ = decay_attention_step(q, k, v, self.log_decay, state)
        return self._project(o)
