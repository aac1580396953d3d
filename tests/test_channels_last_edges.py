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


def check_sizes_refused(device):
    """what one launch's grid and 32-bit chunks do not hold is refused by name, in the call and at the C entries"""
    x = torch.zeros(1, 1, device=device)
    for shape, groups, word in (((65536, 1), 1, "65535"), ((1, (1 << 20) + 1), 1, "1048576"), ((1, 65536), 65536, "65535")):
        with pytest.raises(hip_lib.SaeError, match=word):
            ops.group_norm_act(x.expand(shape), groups)
    lib = hip_lib.get()
    fit = torch.zeros(64, device=device)
    p = fit.data_ptr()
    for n, l, c, groups, word in ((65536, 1, 1, 1, "65535"), (4096, 1 << 31, 1, 1, "2\\^40"), (1, 1 << 41, 1, 1, "2\\^40"),
                                  (2, 2, 6, 4, "groups"), (1, 1, (1 << 20) + 1, 1, "1048576")):
        with pytest.raises(hip_lib.SaeError, match=word):
            lib.call("group_norm_act", p, None, None, p, p, p, None, None, n, l, c, groups, 1e-5, 0, 0.2, 1.0, 0, p, 64, None)
        with pytest.raises(hip_lib.SaeError, match=word):
            lib.call("group_norm_act_bwd", p, p, None, None, p, p, None, None, p, None, None, n, l, c, groups, 0, 0.2, 1.0, 0, p, 64, None)
        assert lib.query("group_norm_act_workspace", n, l, c, groups, 0, 1) == 0
    with pytest.raises(hip_lib.SaeError, match="eps"):
        lib.call("group_norm_act", p, None, None, p, p, p, None, None, 1, 1, 1, 1, -1.0, 0, 0.2, 1.0, 0, p, 64, None)


def check_linear_refused(device):
    """a bias of another length, which the kernel would read past its end, and tensors on two devices"""
    x, w = K.seeded((6, 8), 1).to(device), K.seeded((5, 8), 2).to(device)
    elsewhere = torch.empty(5, 8, device="meta")
    for call in (ops.linear8, ops.linear):
        for args in ((x, w, torch.zeros(4, device=device)), (x, w, torch.zeros(6, device=device)), (x, w, torch.zeros(1, device=device)),
                     (x, w, torch.zeros(5, 5, device=device)), (x, elsewhere), (x, w, elsewhere[:, 0]), (x[:, :7], w), (x, w[:, :7])):
            with pytest.raises(hip_lib.SaeError):
                call(*args)
        assert call(x, w, torch.zeros(5, device=device)).shape == (6, 5)
    for args in ((torch.zeros((), device=device), w), (x, w[0]), (x, w[None])):
        with pytest.raises(hip_lib.SaeError):
            ops.linear8(*args)


CHECKS = [check_frozen_parameters, check_forward_mode, check_negative_views, check_shared, check_linear8_bias_alone]


@pytest.mark.parametrize("check", CHECKS + [check_other_layouts, check_sizes_refused, check_linear_refused], ids=lambda f: f.__name__[6:])
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


# ---- the norm's kernels on both sides of every choice between them, against 64 bits --------------------------------------------

def norm_near(device, dtype, shape, act, checkpoint, mean=0.5, count=64, affine=True):
    """group_norm_act and its backward against the formulas in 64 bits on the same device.  count: a thread's rows, the steps of
    its work-group's fold and the roundings behind -- what is added in fp32 one after the other (records are added in 64 bits)"""
    n, space, c, groups = shape
    full, slope = (n, c) + tuple(space), 0.2
    wide = (1, c) + (1,) * len(space)
    x = ((K.seeded(full, 10) + mean) * (0.5 + K.seeded((c,), 11).abs()).view(wide)).to(dtype).to(device)
    gy = K.seeded(full, 12, dtype, 0.02, 0.1).to(device)
    x, gy = (t.movedim(1, -1).contiguous().movedim(-1, 1) for t in (x, gy))
    leaves = [x.requires_grad_()]
    if affine:
        leaves += [(1 + 0.3 * K.seeded((c,), 13)).to(device).requires_grad_(), (0.2 * K.seeded((c,), 14)).to(device).requires_grad_()]
    y = ops.group_norm_act(*[leaves[0], groups] + leaves[1:], activation=act, negative_slope=slope, checkpoint=checkpoint)
    grads = torch.autograd.grad(y, leaves, gy)
    x = x.detach()
    kept = ops.checkpoint8(x.movedim(1, -1)).dequantize().movedim(-1, 1) if checkpoint else x

    split = lambda t: t.double().reshape(n, groups, c // groups, -1)
    x64, k64, g64 = split(x), split(kept), split(gy)
    w, b = ((t.detach().double().view(1, groups, -1, 1) for t in leaves[1:]) if affine else
            (torch.ones((), dtype=torch.float64, device=device), torch.zeros((), dtype=torch.float64, device=device)))
    scale = 2 ** 0.5 if act == "lrelu" else 1.0
    over = lambda t: t.mean((2, 3), keepdim=True)
    mu = over(x64)
    rstd = (over((x64 - mu) ** 2) + 1e-5) ** -0.5
    e = K.E32
    z = (x64 - mu) * rstd * w + b
    offset = mu.abs() * rstd                                    # the mean is rounded to fp32
    # the variance: sums of (x - x0)^2, off by `count` steps of a sum at most (2 + the distance of x0)^2 larger; rstd by half of that
    spread = count * e * (2 + ((x64 - mu).abs() * rstd).amax((2, 3), keepdim=True)) ** 2
    ey = scale * ((16 * e + spread) * w.abs() * (x64 - mu).abs() * rstd + 16 * e * (w.abs() * offset + b.abs()) + 8 * e) * (1 + z.abs())
    xh = (k64 - mu) * rstd
    zk = xh * w + b
    dz = g64 * scale * K.act_slope64(zk, act, slope)
    ez = (16 * e + spread) * w.abs() * xh.abs() + 16 * e * (w.abs() * offset + b.abs())
    ed = (g64 * scale).abs() * (16 * e * (1 + zk.abs()) + (ez if act == "silu" else 0.0))
    if act == "lrelu":                                          # on either side of the kink
        ed = ed + torch.where(zk.abs() <= ez, (1 - slope) * (g64 * scale).abs(), torch.zeros_like(ed))
    exh = (8 * e + spread) * xh.abs() + 8 * e * offset
    wd = w * dz
    m1, m2 = over(wd), over(wd * xh)
    em1 = over(w.abs() * ed) + count * e * over(wd.abs())
    em2 = over(w.abs() * ed * xh.abs() + wd.abs() * exh) + count * e * over((wd * xh).abs())
    egx = rstd * (w.abs() * ed + em1 + exh * m2.abs() + xh.abs() * em2 + (8 * e + spread) * (wd.abs() + m1.abs() + (xh * m2).abs()))
    total = lambda t: t.sum((0, 3)).view(-1)
    u = K.half_step(dtype)
    checks = [("y", y.detach(), scale * K.act64(z, act, slope), ey, u), ("gx", grads[0], rstd * (wd - m1 - xh * m2), egx, u)]
    if affine:
        checks += [("gw", grads[1], total(dz * xh), total(ed * xh.abs() + dz.abs() * exh + count * e * (dz * xh).abs()), e),
                   ("gb", grads[2], total(dz), total(ed + count * e * dz.abs()), e)]
    for name, got, want, bound, u in checks:
        off = (got.double().reshape(want.shape) - want).abs()
        bound = bound * (1 + u) + u * want.abs() + torch.finfo(dtype).smallest_normal * u
        assert (off <= bound).all(), (name, shape, act, checkpoint, float((off / bound).max()))


# one launch; folded totals in both directions; three launches; more channels than are folded, wide groups, one group, ragged channels
# and groups; sizes on both sides of the one-launch rule (10 MB forward, 4 MB backward)
BORDERS = [(2, (64, 64), 512, 32), (4, (128, 128), 128, 32), (3, (33, 65), 100, 20), (5, (17, 129), 72, 8), (2, (128, 128), 64, 1),
           (2, (40, 50), 1030, 2), (1, (300, 301), 48, 2), (16, (31, 33), 128, 32), (16, (32, 32), 128, 32), (8, (70, 71), 64, 8),
           (2, (9, 9), 2048, 4), (1, (200, 200), 5, 5), (40, (3, 5), 512, 512), (6, (90, 90), 96, 3), (2, (16, 16), 128, 2),
           (2, (16, 16), 512, 1), (4, (15, 16), 256, 16),
           (1, (4, 4), 512, 4), (1, (8, 8), 128, 2), (8, (8, 8), 256, 8), (8, (8, 9), 250, 5)]


@pytest.mark.parametrize("dtype", sorted(K.TYPES))
def test_norm_near_emulated(emu_lib, dtype, monkeypatch):
    """the same check on the sources, each form of launch at small sizes"""
    with backend(emu_lib):
        for one, fold in (("1", "1"), ("0", "1"), ("0", "0")):
            monkeypatch.setenv("SAE_GN_ONE_LAUNCH", one)
            monkeypatch.setenv("SAE_GN_FOLD", fold)
            for act, checkpoint, mean in (("silu", False, 0.5), ("lrelu", True, -3.0), ("none", False, 100.0)):
                norm_near("cpu", K.TYPES[dtype], (2, (13, 27), 40, 4), act, checkpoint, mean, affine=act != "none")


def test_wide_groups_take_more_launches(emu_lib):
    """the backward pass in one launch is for groups that one thread adds up: with a workspace (records of chunks) from 17 channels"""
    for c, groups, one in ((512, 32, True), (512, 30, None), (512, 16, False), (128, 1, False), (34, 2, False), (32, 2, True)):
        if one is None:
            assert emu_lib.query("group_norm_act_workspace", 1, 16, c, groups, 0, 1) == 0        # (no such shape)
        else:
            assert (emu_lib.query("group_norm_act_workspace", 1, 16, c, groups, 0, 1) == 0) == one, (c, groups)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", BORDERS, ids=lambda s: "n%d_%s_c%d_g%d" % (s[0], "x".join(map(str, s[1])), s[2], s[3]))
@pytest.mark.parametrize("dtype", sorted(K.TYPES))
def test_gpu_norm_near(dtype, shape):
    norm_near("cuda:0", K.TYPES[dtype], shape, "silu", False)
    norm_near("cuda:0", K.TYPES[dtype], shape, "silu", True, mean=-3.0)
    norm_near("cuda:0", K.TYPES[dtype], shape, "lrelu", False, mean=0.0)
    norm_near("cuda:0", K.TYPES[dtype], shape, "none", True, mean=100.0, affine=False)


# ---- infinities and NaN at every tile height of the weight gradient ------------------------------------------------------------

def check_wgrad_not_finite(device, dtype, shape):
    """single values that are not finite, in gy and in x, at both ends and in the middle of the rows: every output that does not
    meet one is as near as ever, every other one the infinity or NaN that IEEE arithmetic gives"""
    rows, c, out = shape
    x, gy = K.seeded((rows, c), 1, dtype, 0.2), K.seeded((rows, out), 2, dtype, 0.0, 0.3)
    for i, value in enumerate((float("inf"), float("-inf"), float("nan"))):
        gy[(0, rows // 2, rows - 1)[i], (5 + 61 * i) % out] = value
    gy[rows // 3, 0], gy[rows // 3 + 1, 0] = float("inf"), float("-inf")
    x[rows // 2, c - 1], x[rows - 1, 0] = float("nan"), float("inf")       # whole blocks of 32 channels
    kept = ops.checkpoint8(x.to(device))
    gw, gb = ops.linear_weight_grad8(gy.to(device), kept)
    v, g = kept.dequantize().double(), gy.to(device).double().t().contiguous()
    for got, want, size in ((gw.double(), g @ v, g.abs() @ v.abs()), (gb.double(), g.sum(1), g.abs().sum(1))):
        fine, u = torch.isfinite(want), K.half_step(dtype)
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want))
        assert torch.equal(got[torch.isinf(want)], want[torch.isinf(want)]) and not fine.all()
        assert c <= 64 or fine.any()                                       # (of two blocks none is left)
        off, bound = (got - want).abs(), 2 * K.E32 * (rows + 32) * size * (1 + u) + u * want.abs()
        assert (off <= bound)[fine].all()


@pytest.mark.parametrize("tile", [64, 128, 256])
@pytest.mark.parametrize("dtype", sorted(K.TYPES))
def test_wgrad_not_finite_emulated(emu_lib, dtype, tile, monkeypatch):
    monkeypatch.setenv("SAE_WG_TILE", str(tile))
    with backend(emu_lib):
        for shape in ((70, 130, 300), (330, 64, 140)):
            check_wgrad_not_finite("cpu", K.TYPES[dtype], shape)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(300, 130, 70), (40000, 130, 100), (40000, 200, 300), (33000, 100, 2048)], ids=lambda s: "r%d_c%d_o%d" % s)
@pytest.mark.parametrize("dtype", sorted(K.TYPES))
def test_gpu_wgrad_not_finite(dtype, shape):
    """sizes that take each tile height by themselves"""
    check_wgrad_not_finite("cuda:0", K.TYPES[dtype], shape)


# ---- the framework's own layers inside the context ------------------------------------------------------------------------------

def check_layers_in_context(device):
    """with trainable weights too the input gradient of a layer is the plain one bit for bit (weights as they are, masks by sign),
    and the weight gradient of a product is the one at what is kept of its input, bit for bit"""
    for name, layer, params, shape in _layers(device):
        x, kept = K.seeded(shape, 3).to(device).requires_grad_(), None
        both = []
        for on in (False, True):
            with ops.activation_checkpoints8(least=64, enabled=on):
                y = layer(x)
            both.append(torch.autograd.grad(y, x, K.seeded(y.shape, 4).to(device))[0])
        assert torch.equal(*both), name
        if name in ("ConvLayer", "ResBlock"):
            continue
        h = x.detach() * 1.0
        width = next((w for w in (4096, 512, 64, 32) if h.numel() % w == 0), h.numel())
        kept = ops.checkpoint8(h.reshape(-1, width)).dequantize().view(h.shape)
        gy = K.seeded(y.shape, 5).to(device)
        with ops.activation_checkpoints8(least=64):
            y = layer(h)
        got = torch.autograd.grad(y, params[0], gy)[0]
        if name == "EqualLinear":                               # (the mask is that of the values before they were kept)
            gy = gy * torch.where(y.detach() > 0, 1.0, 0.2) * 2 ** 0.5
            plain = ops.linear(kept, params[0], None, layer.scale)
        else:
            plain = layer(kept)
        want = torch.autograd.grad(plain, params[0], gy)[0]
        if name == "EqualLinear":
            g = gy.cpu().double()
            size = layer.scale * g.abs().t() @ kept.cpu().double().abs()
            assert ((got - want).cpu().double().abs() <= 2 * 8 * K.E32 * size).all(), name
        else:
            assert torch.equal(got, want), name


IN_LAYERS = [check_layers_in_context]


@pytest.mark.parametrize("check", IN_LAYERS, ids=lambda f: f.__name__[6:])
def test_layers_emulated(emu_lib, check):
    with backend(emu_lib):
        check("cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("check", IN_LAYERS, ids=lambda f: f.__name__[6:])
def test_gpu_layers(check):
    check("cuda:0")
