"""The channels-last operators at their edges: frozen weights, shared and foreign tensors inside activation_checkpoints8, forward-mode
differentiation, small gradients, the sizes on both sides of every choice between kernels."""
import pytest
import torch
from torch.autograd import forward_ad

import channels_last_cases as K
from parity_common import backend
from swapping_autoencoder_pytorch_amd import hip_lib
from swapping_autoencoder_pytorch_amd import stylegan2_layers as layers
from swapping_autoencoder_pytorch_amd import stylegan2_op as ops


def _layers(device):
    """(name, layer of at least 4096 weights, input's shape) of the framework's own layers and operators"""
    torch.manual_seed(7)
    conv, matrix = (torch.nn.Parameter(torch.randn(s).to(device)) for s in ((64, 16, 3, 3), (64, 144)))
    made = [("conv2d", lambda x: ops.conv2d(x, conv, padding=1), [conv], (2, 16, 9, 9)),
            ("linear", lambda x: ops.linear(x, matrix), [matrix], (5, 144)),
            ("linear of a view", lambda x: ops.linear(x, conv.view(64, 144)), [conv], (5, 144))]
    for name, layer, shape in (("EqualLinear", layers.EqualLinear(96, 64, activation="fused_lrelu"), (5, 96)),
                               ("EqualConv2d", layers.EqualConv2d(32, 32, 3, padding=1), (2, 32, 8, 8)),
                               ("ConvLayer", layers.ConvLayer(32, 32, 3), (2, 32, 8, 8)),
                               ("ResBlock", layers.ResBlock(32, 32), (2, 32, 16, 16))):
        layer = layer.to(device)
        made.append((name, layer, list(layer.parameters()), shape))
    return made


def check_frozen_parameters(device):
    """a Parameter is kept as it is whether it requires a gradient or not: the input gradient through a frozen layer is the plain one
    bit for bit (what is packed besides are the layer's own activations, read by their signs alone)"""
    for name, layer, params, shape in _layers(device):
        x = K.seeded(shape, 3).to(device)
        for p in params:
            p.requires_grad_(False)
        grads = []
        for on in (False, True):
            leaf = x.clone().requires_grad_()
            with ops.activation_checkpoints8(least=64, enabled=on):
                y = layer(leaf)
            grads.append(torch.autograd.grad(y, leaf, K.seeded(y.shape, 4).to(device))[0])
        assert torch.equal(*grads), name


def check_forward_mode(device):
    """a tangent is refused, as by every custom function of the framework, never dropped; inside a level without tangents nothing
    changes"""
    x, w = K.seeded((2, 8, 3), 1).to(device), K.seeded((8,), 2).to(device)
    want = ops.group_norm_act(x, 2, w)
    with forward_ad.dual_level():
        for args in ((forward_ad.make_dual(x, torch.ones_like(x)), 2, w), (x, 2, forward_ad.make_dual(w, torch.ones_like(w))),
                     (x, 2, None, forward_ad.make_dual(w, torch.ones_like(w)))):
            with pytest.raises(NotImplementedError):
                ops.group_norm_act(*args)
            with pytest.raises(NotImplementedError), torch.no_grad():
                ops.group_norm_act(*args)
        assert torch.equal(ops.group_norm_act(x, 2, w), want)


def check_other_layouts(device):
    """a saved tensor without strides stays as it is"""
    x = K.seeded((40, 40), 1).to(device).requires_grad_()
    a = (K.seeded((40, 40), 2) * (K.seeded((40, 40), 3) > 0)).to(device)
    for sparse in (a.to_sparse(), a.to_sparse_csr()):
        with ops.activation_checkpoints8(least=64):
            y = sparse @ (x * 1.0)
        gx, = torch.autograd.grad(y, x, torch.ones_like(y))
        assert torch.allclose(gx, a.sum(0)[:, None].expand(40, 40), rtol=0, atol=40 * K.E32 * 40)


def check_negative_views(device):
    """the imaginary part of a conjugate is a view with its sign in a flag: read with the sign"""
    z = torch.complex(K.seeded((1, 1), 1), K.seeded((1, 1), 2)).to(device)
    x = z.conj().imag
    assert x.is_neg() and x.is_contiguous()
    wide = torch._neg_view(K.seeded((2, 4, 8, 8), 3).to(device).contiguous(memory_format=torch.channels_last))
    for t in (x, wide.movedim(1, -1)):
        assert torch.equal(ops.checkpoint8(t).dequantize(), ops.checkpoint8(t.resolve_neg().clone()).dequantize())
    assert torch.equal(ops.group_norm_act(wide, 2), ops.group_norm_act(wide.resolve_neg(), 2))
    rows = wide.reshape(-1, 8)
    kept = ops.checkpoint8(rows)
    assert torch.equal(ops.linear_weight_grad8(rows, kept)[0], ops.linear_weight_grad8(rows.resolve_neg(), kept)[0])


CHECKS = [check_frozen_parameters, check_forward_mode, check_negative_views]


@pytest.mark.parametrize("check", CHECKS + [check_other_layouts], ids=lambda f: f.__name__[6:])
def test_emulated(emu_lib, check):
    with backend(emu_lib):
        check("cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("check", CHECKS, ids=lambda f: f.__name__[6:])
def test_gpu(check):
    check("cuda:0")
