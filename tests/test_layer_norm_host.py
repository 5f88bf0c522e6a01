"""What `layer_norm` makes of autograd's modes, without a GPU: the launch is replaced by the oracle, which like the
kernels fills memory that no torch operation writes."""

import pytest
import torch
from torch.autograd import forward_ad

from axonn_amd import ops
from axonn_amd.intra_layer import LayerNorm, layer_norm
from oracle import layer_norm as ol


@pytest.fixture
def launches(monkeypatch):
    """The calls of `ops.layer_norm_fwd`, answered by the oracle."""
    calls = []

    def forward(x, weight=None, bias=None, eps=1e-5, residual=None, save=True):
        calls.append(save)
        f = lambda t: None if t is None else t.detach().numpy()  # noqa: E731
        h = f(x) if residual is None else f(x) + f(residual)
        out = [torch.empty_like(x), torch.empty_like(x), torch.empty(len(x)), torch.empty(len(x))]
        y, mean, rstd = ol.forward(h, f(weight), f(bias), eps)
        for t, value in zip(out, (y, h, mean, rstd)):
            t.numpy()[...] = value
        return (out[0], None if residual is None else out[1], *(out[2:] if save else (None, None)))

    monkeypatch.setattr(ops, "layer_norm_fwd", forward)
    return calls


@pytest.mark.parametrize("which", ["x", "residual", "weight", "bias"])
@pytest.mark.parametrize("gradients", [True, False])
def test_forward_mode_derivatives_are_refused(launches, which, gradients):
    """Not dropped: a result without a tangent would be a derivative of zero."""
    args = dict(x=torch.randn(3, 8), residual=torch.randn(3, 8), weight=torch.ones(8), bias=torch.zeros(8))
    with torch.set_grad_enabled(gradients), forward_ad.dual_level():
        plain = layer_norm(normalized_shape=8, **args)     # (none of them has a tangent: as outside)
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError, match="jvp"):
            layer_norm(normalized_shape=8, **args)
    with torch.no_grad():
        args[which] = forward_ad.unpack_dual(args[which]).primal
        assert all(torch.equal(a, b) for a, b in zip(plain, layer_norm(normalized_shape=8, **args)))


def test_a_layer_without_gradients_keeps_no_statistics(launches):
    layer, x = LayerNorm(8), torch.randn(3, 8)
    with torch.no_grad():
        layer(x), layer(x, x)
    assert launches == [False, False]
    layer(x)
    assert launches[2:] == [True]


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("gradients", [True, False])
@pytest.mark.parametrize("with_residual", [False, True])
def test_a_trace_computes_what_the_layer_does(launches, gradients, with_residual):
    """The call itself is in the graph, whatever mode it is recorded in and run in, and not the memory it filled."""
    layer = LayerNorm(8)
    with torch.no_grad():
        layer.weight.mul_(1.5)
    operands = lambda: tuple(torch.randn(3, 8) for _ in range(1 + with_residual))  # noqa: E731
    with torch.set_grad_enabled(gradients):
        traced = torch.jit.trace(layer, operands(), check_trace=False)
    for again in (False, True, False):
        args = operands()
        with torch.set_grad_enabled(again):
            got, want = traced(*args), layer(*args)
        for a, b in zip(*((got, want) if with_residual else ((got,), (want,)))):
            assert torch.equal(a, b) and a.requires_grad == again


@pytest.mark.parametrize("which", ["x", "residual", "weight", "bias"])
def test_autocast_leaves_64_bits_as_they_are(launches, monkeypatch, which):
    """Autocast widens 16 bits to 32; 64 bits, which the kernels do not have, reach their check of types and are not
    made 32 on the way."""
    seen = []
    forward = ops.layer_norm_fwd
    monkeypatch.setattr(ops, "layer_norm_fwd", lambda x, weight, bias, eps, residual=None, save=True: (
        seen.append([t.dtype for t in (x, residual, weight, bias)]), forward(x, weight, bias, eps, residual, save))[1])
    monkeypatch.setattr(torch, "is_autocast_enabled", lambda *device: True)
    args = dict(x=torch.randn(3, 8).half(), residual=torch.randn(3, 8).bfloat16(), weight=torch.ones(8), bias=torch.zeros(8).half())
    for gradients in (True, False):
        with torch.set_grad_enabled(gradients):
            layer_norm(normalized_shape=8, **args)
            assert seen.pop() == [torch.float32] * 4
            layer_norm(normalized_shape=8, **{**args, which: args[which].double()})
            assert seen.pop() == [torch.float64 if w == which else torch.float32 for w in args]
