"""The channels-last operators at their edges: frozen weights, shared and foreign tensors inside activation_checkpoints8, forward-mode
differentiation, small gradients, the sizes on both sides of every choice between kernels."""
import contextlib

import pytest
import torch
from torch.autograd import forward_ad
from torch.utils._python_dispatch import TorchDispatchMode

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


def _packs(run):
    """run() and how often it packed"""
    lib = hip_lib.get()
    plain, names = lib.call, []

    def call(name, *args):
        names.append(name)
        return plain(name, *args)
    lib.call = call
    try:
        return run(), names.count("checkpoint8_pack")
    finally:
        del lib.call


def kept_values(t):
    """what the context keeps of a contiguous t, in 64 bits"""
    return K.plain_codes(t.detach().cpu().reshape(-1, 64))[2].view(t.shape)


def check_shared(device):
    """nodes that save the same tensor share one checkpoint; a tensor that was written in between, another view and new values in
    the same memory have their own.  Every gradient is a sum of at most three products of kept values."""
    x = K.seeded((64, 64), 1).to(device).requires_grad_()
    gz = K.seeded((64, 64), 2).to(device)
    plain = {}

    def near(got, want, size):
        assert ((got.cpu().double() - want).abs() <= 8 * K.E32 * size).all()

    def shared():
        with ops.activation_checkpoints8(least=64):
            h = x * 1.0
            s = torch.sigmoid(h)
            y = h * h
            z = s * y
        plain.update(h=h, s=s, y=y)
        return z
    z, packs = _packs(shared)
    assert packs == 3                                # h, s, y: saved five times
    h, s, y = (kept_values(plain[n]) for n in "hsy")
    g = gz.cpu().double()
    gx, = torch.autograd.grad(z, x, gz)
    near(gx, 2 * g * s * h + g * y * s * (1 - s), 2 * (g * s * h).abs() + (g * y * s).abs() * (1 + s.abs()))

    def written():
        with ops.activation_checkpoints8(least=64):
            w = x.detach() * 1.0
            a = x * w                                # (x is a leaf: only w is kept)
            first = w.clone()
            w.mul_(-3.0)
            b = x * w
        return a, b, first, w
    (a, b, first, w), packs = _packs(written)
    assert packs == 2
    for out, want in ((a, first), (b, w)):
        near(torch.autograd.grad(out, x, gz)[0], g * kept_values(want), (g * kept_values(want)).abs())

    def views():
        with ops.activation_checkpoints8(least=64):
            w = x.detach() * 1.0
            return [x[:32] * w[:32], x[32:] * w[32:], x * w, x.t() * w.t()], w
    (outs, w), packs = _packs(views)
    assert packs == 4
    parts = [torch.cat([g[:32], g[:32]]) * kept_values(w), g * kept_values(w), g.t() * kept_values(w)]
    near(sum(torch.autograd.grad(o, x, gz[:o.shape[0]] if i < 2 else gz)[0] for i, o in enumerate(outs)), sum(parts),
         sum(t.abs() for t in parts))

    # freed memory that comes back with other values
    with ops.activation_checkpoints8(least=64):
        outs = [x * (x.detach() * float(i)) for i in range(1, 9)]
    for i, o in enumerate(outs):
        want = g * kept_values(x.detach() * float(i + 1))
        near(torch.autograd.grad(o, x, gz)[0], want, want.abs())


class _Reductions(TorchDispatchMode):
    """torch's own sums, which put nodes into a captured graph that do not replay reliably"""

    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        if func.overloadpacket in (torch.ops.aten.sum, torch.ops.aten.mean):
            self.seen.append(func)
        return func(*args, **(kwargs or {}))


def check_linear8_bias_alone(device):
    """the bias gradient beside a frozen weight and under input_grads_only: the framework's own sum of the rows"""
    for rows in (0, 1, 70, 5000):
        x, w = K.seeded((rows, 36), 1).to(device), K.seeded((20, 36), 2).to(device)
        b, gy = K.seeded((20,), 3).to(device).requires_grad_(), K.seeded((rows, 20), 4).to(device)
        g = gy.cpu().double()
        for frozen in (True, False):
            y = ops.linear8(x, w if frozen else w.clone().requires_grad_(), b)
            with _Reductions() as torchs, (contextlib.nullcontext() if frozen else ops.input_grads_only()):
                gb, = torch.autograd.grad(y, b, gy)
            assert not torchs.seen
            assert ((gb.cpu().double() - g.sum(0)).abs() <= 2 * K.E32 * (rows + 32) * g.abs().sum(0)).all()


CHECKS = [check_frozen_parameters, check_forward_mode, check_negative_views, check_shared, check_linear8_bias_alone]


@pytest.mark.parametrize("check", CHECKS + [check_other_layouts], ids=lambda f: f.__name__[6:])
def test_emulated(emu_lib, check):
    with backend(emu_lib):
        check("cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("check", CHECKS, ids=lambda f: f.__name__[6:])
def test_gpu(check):
    check("cuda:0")


@pytest.mark.gpu
def test_gpu_context_memory():
    """what the context holds of an activation that two nodes save: 33 bytes for 32 values, once"""
    for dtype, share in ((torch.float32, 33 / 128), (torch.bfloat16, 33 / 64)):
        x = torch.randn(64, 1 << 18, device="cuda").to(dtype).requires_grad_()
        size = x.numel() * x.element_size()
        held = []
        for on in (False, True):
            torch.cuda.synchronize()
            before = torch.cuda.memory_allocated()
            with ops.activation_checkpoints8(enabled=on):
                h = x * 1.0
                out = (torch.sigmoid(h) * (h * h)).sum()             # h three times, its sigmoid twice, the square once
                del h
            torch.cuda.synchronize()
            held.append((torch.cuda.memory_allocated() - before) / size)
            del out
        assert abs(held[0] - 3) < 0.01 and abs(held[1] - 3 * share) < 0.01, (dtype, held)


@pytest.mark.gpu
def test_gpu_shared_on_two_streams_and_captured():
    """a tensor that is saved eagerly, on another stream and inside a capture of the same block: each replay reads what the tensor
    holds then (the leaves of the captured and of the eager nodes are not the same)"""
    make = lambda seed: K.seeded((256, 512), seed).cuda()
    h, gy = make(1), make(2)
    leaves = [make(3).requires_grad_() for _ in range(3)]
    kept = lambda t: ops.checkpoint8(t).dequantize()
    side, warm = torch.cuda.Stream(), torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm), ops.activation_checkpoints8(least=64):
        torch.autograd.grad((leaves[2] * h) * h, leaves[2], gy)
    torch.cuda.current_stream().wait_stream(warm)
    graph = torch.cuda.CUDAGraph()
    with ops.activation_checkpoints8(least=64):
        eager = leaves[0] * h
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = leaves[1] * h
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out, = torch.autograd.grad((leaves[2] * h) * h, leaves[2], gy)
    want = kept(h) * gy
    assert torch.equal(torch.autograd.grad(eager, leaves[0], gy)[0], want)
    assert torch.equal(torch.autograd.grad(other, leaves[1], gy)[0], want)
    for seed in (4, 5, 6):
        h.copy_(make(seed))
        graph.replay()
        torch.cuda.synchronize()
        got, want = out.clone(), gy * kept(h) * kept(h)
        torch.cuda.synchronize()
        assert torch.equal(got, want), seed


# ---- small gradients, and values next to the ends of a type's range ------------------------------------------------------------

def _wgrad_near(device, x, gy, dtype, less):
    """linear_weight_grad8 against 64 bits.  Every fp32 addition is off by one step at most; outputs are rounded once, at least to
    the last place of the type's subnormals; `less`: how far a value of gy may be off before it is multiplied"""
    kept = ops.checkpoint8(x.to(device))
    gw, gb = (t.cpu().double() for t in ops.linear_weight_grad8(gy.to(device), kept))
    v, g, rows = K.plain_codes(x)[2], gy.double(), x.shape[0]
    u, last = K.half_step(dtype), torch.finfo(dtype).smallest_normal * K.half_step(dtype)
    for got, want, size, slack in ((gw, g.t() @ v, g.abs().t() @ v.abs(), less * v.abs().sum(0)),
                                   (gb, g.sum(0), g.abs().sum(0), torch.zeros(()))):
        bound = (2 * K.E32 * (rows + 32) * size + rows * 2.0 ** -149 + slack) * (1 + u) + u * want.abs() + last
        assert ((got - want).abs() <= bound).all(), float(((got - want).abs() / bound).max())


def check_small_gradients(device, dtype, scale):
    for rows, c, out in ((70, 40, 33), (300, 64, 129)):
        x, gy = K.seeded((rows, c), 1, dtype, 0.2), K.seeded((rows, out), 2, dtype, 0.0, scale)
        # f32: pieces of bf16, whose last place is 2^-133: the two lower ones are cut there, less than a place each
        _wgrad_near(device, x, gy, dtype, 2.0 ** -132 if dtype == torch.float32 else 0.0)


SMALL = [("f16", 1e-3), ("f16", 1e-5), ("f16", 3e-7), ("bf16", 1e-20), ("bf16", 1e-38), ("f32", 1e-20), ("f32", 1e-32), ("f32", 1e-36),
         ("f32", 1e-38), ("f32", 1e-40)]


@pytest.mark.parametrize("dtype,scale", SMALL)
def test_small_gradients_emulated(emu_lib, dtype, scale):
    with backend(emu_lib):
        check_small_gradients("cpu", K.TYPES[dtype], scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,scale", SMALL)
def test_gpu_small_gradients(dtype, scale):
    check_small_gradients("cuda:0", K.TYPES[dtype], scale)
