"""group_norm_act, checkpoint8, linear_weight_grad8 / linear8 and activation_checkpoints8 against plain 64-bit forms: the kernel
sources on the emulator (CPU) and the built library (``-m gpu``); their refusals (CPU)."""
import pytest
import torch

import channels_last_cases as K
from parity_common import backend
from swapping_autoencoder_pytorch_amd import hip_lib
from swapping_autoencoder_pytorch_amd import stylegan2_op as ops

TYPES = sorted(K.TYPES)
ACTS = ["none", "lrelu", "silu"]


def norm_id(s):
    return "n%d_%s_c%d_g%d" % (s[0], "x".join(map(str, s[1])) or "flat", s[2], s[3])


# ---- refusals and what needs no kernel (first: a call that should not run must not) -------------------------------------------

def test_refusals(emu_lib):
    x = torch.randn(2, 8, 3, 3)
    w = torch.ones(8)
    with backend(emu_lib):
        for bad in (dict(num_groups=3), dict(num_groups=0), dict(num_groups=2, activation="relu"), dict(num_groups=2, eps=-1.0),
                    dict(num_groups=2, weight=torch.ones(7)), dict(num_groups=2, weight=w.double()),
                    dict(num_groups=2, bias=torch.ones(8, dtype=torch.bfloat16)), dict(num_groups=2, eps=float("nan"))):
            with pytest.raises(hip_lib.SaeError):
                ops.group_norm_act(x, **bad)
        for t in (x.double(), x.int(), torch.randn(5), torch.randn(2, 0, 3)):
            with pytest.raises(hip_lib.SaeError):
                ops.group_norm_act(t, 1)
        for t in (x.double(), torch.randn(()), torch.randn(3, 0)):
            with pytest.raises(hip_lib.SaeError):
                ops.checkpoint8(t)
        kept = ops.checkpoint8(torch.randn(4, 40))
        for gy in (torch.randn(5, 3), torch.randn(4, 3).bfloat16(), torch.randn(4, 0)):
            with pytest.raises(hip_lib.SaeError):
                ops.linear_weight_grad8(gy, kept)
        good = (kept.codes, kept.scales, 40, torch.float32)
        for at, value in ((0, kept.codes[:, :32]), (0, kept.codes.float()), (0, kept.codes[:3]), (1, kept.scales.t()),
                          (1, kept.scales[:1]), (1, kept.scales.int()), (2, 33 + 32), (2, 32), (2, 0), (3, torch.float64)):
            bad = list(good)
            bad[at] = value
            with pytest.raises(hip_lib.SaeError):
                ops.Checkpoint8(*bad)
        with pytest.raises(hip_lib.SaeError):
            ops.Checkpoint8(*good, shape=(3, 40))


def test_entry_points_refuse(emu_lib, monkeypatch):
    """the C entry points' own checks: null tensors, unknown codes, misalignment, short workspaces"""
    monkeypatch.setenv("SAE_GN_ONE_LAUNCH", "0")     # the form that needs a workspace
    x = torch.randn(4, 16)
    y, w = torch.empty_like(x), torch.ones(16)
    stats = torch.empty(2, 8)
    codes, scales = torch.empty(4, 32, dtype=torch.int8), torch.empty(1, 4, dtype=torch.uint8)
    n = emu_lib.query("group_norm_act_workspace", 2, 2, 16, 4, 0, 0)
    nb = emu_lib.query("group_norm_act_workspace", 2, 2, 16, 4, 0, 1)
    assert n > 0 and nb > 0
    ws = torch.empty(max(n, nb), dtype=torch.uint8)
    p = lambda t: t.data_ptr()
    good = [p(x), p(w), p(w), p(y), p(stats[0]), p(stats[1]), p(codes), p(scales), 2, 2, 16, 4, 1e-5, 1, 0.2, 1.0, 0, p(ws), n, None]
    emu_lib.call("group_norm_act", *good)
    for at, value in ((0, None), (3, None), (4, None), (6, None), (8, -1), (10, 15), (11, 0), (12, -1.0), (13, 3), (16, 5), (17, None),
                      (18, n - 1), (0, p(x) + 4), (3, p(y) + 4), (8, 65536)):
        bad = list(good)
        bad[at] = value
        with pytest.raises(hip_lib.SaeError):
            emu_lib.call("group_norm_act", *bad)
    good = [p(x), p(x), None, None, p(stats[0]), p(stats[1]), p(w), p(w), p(y), p(w), p(w), 2, 2, 16, 4, 1, 0.2, 1.0, 0, p(ws), nb, None]
    for at, value in ((0, None), (1, None), (2, p(codes)), (4, None), (11, -1), (14, 5), (15, -1), (18, 3), (19, None), (20, nb - 1)):
        bad = list(good)
        bad[at] = value
        with pytest.raises(hip_lib.SaeError):
            emu_lib.call("group_norm_act_bwd", *bad)
    good = [p(x), p(codes), p(scales), 4, 16, 0, None]
    for at, value in ((0, None), (1, None), (2, None), (3, -1), (4, 0), (5, 3), (1, p(codes) + 1), (0, p(x) + 1)):
        bad = list(good)
        bad[at] = value
        for name in ("checkpoint8_pack", "checkpoint8_unpack"):
            args = bad if name.endswith("_pack") and not name.endswith("unpack") else [bad[1], bad[2], bad[0]] + bad[3:]
            with pytest.raises(hip_lib.SaeError):
                emu_lib.call(name, *args)
    rows = 600                                       # several slices: with a workspace
    n = emu_lib.query("linear_wgrad8_workspace", rows, 16, 16, 0)
    assert n > 0 and emu_lib.query("linear_wgrad8_workspace", 4, 16, 16, 0) == 0
    gy, codes, scales = torch.zeros(rows, 16), torch.zeros(rows, 32, dtype=torch.int8), torch.full((1, rows), 127, dtype=torch.uint8)
    wsf, gw = torch.empty(n), torch.empty(16, 16)
    good = [p(gy), p(codes), p(scales), p(gw), None, rows, 16, 16, 1.0, 0, p(wsf), n, None]
    emu_lib.call("linear_wgrad8", *good)
    for at, value in ((0, None), (1, None), (2, None), (3, None), (5, -1), (6, 0), (7, 0), (9, 3), (10, None), (11, n - 1), (1, p(codes) + 4),
                      (0, p(gy) + 2)):
        bad = list(good)
        bad[at] = value
        with pytest.raises(hip_lib.SaeError):
            emu_lib.call("linear_wgrad8", *bad)


def test_no_cpu_path():
    """the product's library takes no host tensors"""
    for call in (lambda: ops.group_norm_act(torch.randn(2, 8, 3), 2), lambda: ops.checkpoint8(torch.randn(2, 8))):
        with pytest.raises(hip_lib.SaeError):
            call()


def test_context_leaves_host_tensors():
    """what the product's library does not take is kept as it is"""
    x = torch.randn(50, 40, requires_grad=True)
    with ops.activation_checkpoints8(least=1):
        y = (x * 1.5) ** 2
    assert torch.equal(torch.autograd.grad(y.sum(), x)[0], 2 * (x.detach() * 1.5) * 1.5)


# ---- values -------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
def test_checkpoint8_emulated(emu_lib, dtype):
    with backend(emu_lib):
        K.check_checkpoint8("cpu", K.TYPES[dtype])


@pytest.mark.parametrize("dtype", TYPES)
def test_oracle_checkpoint8(oracle_lib, dtype):
    with backend(oracle_lib):
        K.check_checkpoint8("cpu", K.TYPES[dtype])


@pytest.mark.parametrize("checkpoint", [False, True], ids=["full", "kept8"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", TYPES)
def test_oracle_norm(oracle_lib, dtype, act, checkpoint):
    with backend(oracle_lib):
        for shape in K.NORM_SHAPES[:6]:
            K.check_norm("cpu", K.TYPES[dtype], shape, act, checkpoint)


@pytest.mark.parametrize("dtype", TYPES)
def test_oracle_wgrad(oracle_lib, dtype):
    with backend(oracle_lib):
        for shape in K.WGRAD_SHAPES[:5]:
            K.check_wgrad("cpu", K.TYPES[dtype], shape, alpha=0.7)


def test_the_formulas_are_autograds():
    """norm64's gradients (from the uncompressed input) against torch's derivative of its forward formula, and both against
    differences"""
    for act in ACTS:
        x = K.seeded((2, 12, 5), 1).double().requires_grad_()
        w, b = (K.seeded((12,), s).double().requires_grad_() for s in (2, 3))
        gy = K.seeded((2, 12, 5), 4).double()

        def forward(x, w, b):
            xg = x.reshape(2, 3, -1)
            xh = ((xg - xg.mean(2, keepdim=True)) * (xg.var(2, unbiased=False, keepdim=True) + 1e-5) ** -0.5).view(2, 12, 5)
            return 1.3 * K.act64(xh * w[:, None] + b[:, None], act, 0.2)
        want = torch.autograd.grad(forward(x, w, b), [x, w, b], gy)
        with torch.no_grad():
            r = K.norm64(x, x, gy, 3, w, b, 1e-5, act, 0.2, 1.3)
            for got, ref in zip((r["gx"].view(2, 12, 5), r["gw"], r["gb"]), want):
                assert torch.allclose(got, ref, rtol=1e-10, atol=1e-12)
            for t, g in zip((x, w, b), want):
                d = K.seeded(t.shape, 7).double()
                args = lambda s: [v + s * d if v is t else v for v in (x, w, b)]
                diff = ((forward(*args(1e-6)) - forward(*args(-1e-6))) * gy).sum() / 2e-6
                assert abs(float(diff - (g * d).sum())) <= 1e-6 * float((g * d).abs().sum())


@pytest.mark.parametrize("shape", K.NORM_SHAPES, ids=norm_id)
@pytest.mark.parametrize("dtype", TYPES)
def test_norm_emulated(emu_lib, dtype, shape):
    with backend(emu_lib):
        for i, act in enumerate(ACTS):
            K.check_norm("cpu", K.TYPES[dtype], shape, act, checkpoint=False, affine=i != 0)
            K.check_norm("cpu", K.TYPES[dtype], shape, act, checkpoint=True, affine=i != 1)


@pytest.mark.parametrize("shape", K.NORM_SHAPES, ids=norm_id)
@pytest.mark.parametrize("dtype", TYPES)
def test_norm_in_three_launches_emulated(emu_lib, dtype, shape, monkeypatch):
    """small groups through the kernels of the large ones (the knob exists in tuning builds only)"""
    monkeypatch.setenv("SAE_GN_ONE_LAUNCH", "0")
    with backend(emu_lib):
        for fold in ("1", "0"):                      # two launches, and with one for the totals
            monkeypatch.setenv("SAE_GN_FOLD", fold)
            K.check_norm("cpu", K.TYPES[dtype], shape, "silu", checkpoint=False)
            K.check_norm("cpu", K.TYPES[dtype], shape, "lrelu", checkpoint=True)
            K.check_norm("cpu", K.TYPES[dtype], shape, "none", checkpoint=False, affine=False)


@pytest.mark.parametrize("shape", K.WGRAD_SHAPES, ids=lambda s: "r%d_c%d_o%d" % s)
@pytest.mark.parametrize("dtype", TYPES)
def test_wgrad_emulated(emu_lib, dtype, shape):
    with backend(emu_lib):
        K.check_wgrad("cpu", K.TYPES[dtype], shape)
        if shape[0] < 60:
            K.check_wgrad("cpu", K.TYPES[dtype], shape, alpha=-0.37, bias=False)


# ---- the operators in use: memory orders, the context, a run of them together, graphs, streams ---------------------------------

def check_memory_orders(device):
    for memory in ("plain", "sliced"):
        for dtype in K.TYPES.values():
            K.check_norm(device, dtype, (2, (5, 7), 24, 3), "silu", memory == "sliced", memory=memory)
    x = K.seeded((6, 10, 50), 3).to(device)
    whole, part = ops.checkpoint8(x), ops.checkpoint8(x[:, 3:, 1:])
    assert torch.equal(part.dequantize(), ops.checkpoint8(x[:, 3:, 1:].contiguous()).dequantize())
    assert whole.shape == x.shape and part.shape == (6, 7, 49) and whole.nbytes == 60 * 66
    gy = K.seeded((60, 22), 4).to(device)
    kept = ops.checkpoint8(K.seeded((60, 40), 5).to(device))
    for view in (gy[:, 2:], gy[:, 1:10], gy.t().contiguous().t()):
        got, want = ops.linear_weight_grad8(view, kept), ops.linear_weight_grad8(view.contiguous().clone(), kept)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def check_empty(device):
    for space in ((), (0,), (4, 0)):
        n = 0 if space == () else 2
        x = torch.randn((n, 8) + space, device=device, requires_grad=True)
        w, b = (torch.randn(8, device=device, requires_grad=True) for _ in range(2))
        for keep in (False, True):
            y = ops.group_norm_act(x, 2, w, b, checkpoint=keep)
            gx, gw, gb = torch.autograd.grad(y, [x, w, b], torch.ones_like(y))
            assert y.shape == gx.shape == x.shape and not gw.any() and not gb.any()
    kept = ops.checkpoint8(torch.randn(0, 40, device=device))
    assert kept.dequantize().shape == (0, 40) and kept.nbytes == 0
    gw, gb = ops.linear_weight_grad8(torch.randn(0, 5, device=device), kept)
    assert gw.shape == (5, 40) and not gw.any() and not gb.any()


def check_not_finite(device):
    """a NaN or infinity stays in its group (norm) and in its block (checkpoint)"""
    x = K.seeded((2, 64, 4, 4), 3)
    x[0, 5, 1, 1], x[1, 40, 0, 0] = float("nan"), float("inf")
    y = ops.group_norm_act(x.to(device), 8, activation="silu").cpu()
    bad = torch.isnan(y.reshape(2, 8, -1))
    assert bad[0, 0].all() and bad[1, 5].all() and int(bad.sum()) == 2 * 8 * 16
    # gw of a weight gradient: rows of channels whose checkpoint is NaN, columns whose gradient is not finite
    x, gy = K.seeded((40, 64), 6), K.seeded((40, 9), 7)
    x[3, 40] = float("nan")
    gy[7, 2], gy[8, 4] = float("inf"), float("-inf")
    gw, gb = (t.cpu() for t in ops.linear_weight_grad8(gy.to(device), ops.checkpoint8(x.to(device))))
    assert torch.isnan(gw[:, 32:]).all() and torch.isfinite(gw[[0, 1, 3, 5, 6, 7, 8], :32]).all()
    assert torch.equal(gw[2, :32], torch.sign(x[7, :32]) * float("inf")) and torch.equal(gw[4, :32], -torch.sign(x[8, :32]) * float("inf"))
    assert gb[2] == float("inf") and gb[4] == float("-inf") and torch.isfinite(gb[[0, 1, 3, 5]]).all()


def check_linear8(device):
    """y and the input gradient are linear's bit for bit, the others are those of the kept input"""
    x, w, b = (K.seeded(s, i).to(device).requires_grad_() for i, s in ((1, (3, 11, 48)), (2, (20, 48)), (3, (20,))))
    gy = K.seeded((3, 11, 20), 4).to(device)
    y, ref = ops.linear8(x, w, b, 0.8), ops.linear(x, w, b, 0.8)
    assert torch.equal(y, ref)
    gx, gw, gb = torch.autograd.grad(y, [x, w, b], gy)
    assert torch.equal(gx, torch.autograd.grad(ref, x, gy)[0])
    kept = K.plain_codes(x.detach().cpu().view(33, 48))[2]
    g = gy.cpu().double().view(33, 20)
    assert ((gw.cpu().double() - 0.8 * g.t() @ kept).abs() <= 2 * K.E32 * 70 * (g.abs().t() @ kept.abs())).all()
    assert ((gb.cpu().double() - g.sum(0)).abs() <= 2 * K.E32 * 70 * g.abs().sum(0)).all()
    frozen = ops.linear8(x, w.detach(), b)
    gx, gb = torch.autograd.grad(frozen, [x, b], gy)
    assert torch.equal(gx, torch.autograd.grad(ops.linear(x, w.detach(), b), x, gy)[0])
    only = torch.autograd.grad(ops.linear8(x.detach(), w), w, gy)[0]
    assert ((only.cpu().double() - g.t() @ kept).abs() <= 2 * K.E32 * 70 * (g.abs().t() @ kept.abs())).all()
    with ops.input_grads_only():
        assert torch.autograd.grad(ops.linear8(x, w, b), [x, w], gy, allow_unused=True)[1] is None
    with torch.no_grad():
        assert torch.equal(ops.linear8(x, w, b, 0.8), ref)


def check_run_together(device):
    """norm + activation -> linear over the maps, both kept in 8 bits, as a training step uses them: the gradients against the
    64-bit forms at the kept values"""
    n, c, h, out = 2, 64, 9, 40
    x = K.seeded((n, c, h, h), 1, mean=0.3).to(device).movedim(1, -1).contiguous().movedim(-1, 1).requires_grad_()
    norm = ops.GroupNormAct(8, c, activation="silu", checkpoint=True).to(device)
    with torch.no_grad():
        norm.weight.copy_(1 + 0.2 * K.seeded((c,), 2))
        norm.bias.copy_(0.2 * K.seeded((c,), 3))
    w, b = K.seeded((out, c), 4).to(device).requires_grad_(), torch.zeros(out, device=device, requires_grad=True)
    y = norm(x)
    z = ops.linear8(y.movedim(1, -1), w, b)
    gz = K.seeded((n, h, h, out), 5).to(device)
    gy, = torch.autograd.grad(z, y, gz, retain_graph=True)            # what the product hands the norm, bit for bit
    grads = torch.autograd.grad(z, [x, norm.weight, norm.bias, w, b], gz)
    kept_y = ops.checkpoint8(y.detach().movedim(1, -1)).dequantize().cpu().double().view(-1, c)
    g = gz.cpu().double().view(-1, out)
    assert ((grads[3].cpu().double() - g.t() @ kept_y).abs() <= 2 * K.E32 * (n * h * h + 32) * (g.abs().t() @ kept_y.abs())).all()
    kept_x = K.plain_codes(x.detach().cpu().movedim(1, -1).reshape(-1, c))[2].view(n, h, h, c).movedim(-1, 1)
    r = K.norm64(x.detach().cpu(), kept_x, gy.cpu(), 8, norm.weight.detach().cpu(), norm.bias.detach().cpu(), 1e-5, "silu", 0.2, 1.0)
    for got, name in zip(grads, ("gx", "gw", "gb")):
        off = (got.cpu().double().reshape(r[name].shape) - r[name]).abs()
        assert (off <= r["e" + name] + K.E32 * r[name].abs()).all(), name


def check_context(device):
    """the framework's own layers inside the context: the same values, the input gradient of a leaky ReLU exact (its mask is a
    sign), weight gradients those of the kept input"""
    x = K.seeded((2, 8, 24, 24), 1).to(device).requires_grad_()
    w = torch.nn.Parameter(K.seeded((16, 8, 1, 1), 2).to(device))
    b = torch.nn.Parameter(K.seeded((16,), 3).to(device))
    gy = K.seeded((2, 16, 24, 24), 4).to(device)

    def step():
        y = ops.fused_leaky_relu(ops.conv2d(x, w), b)
        return (y,) + torch.autograd.grad(y, [x, w, b], gy)
    plain = step()
    with ops.activation_checkpoints8(enabled=False):
        same = step()
    with ops.activation_checkpoints8(least=1 << 40):
        small = step()
    with ops.activation_checkpoints8(least=64):
        kept = step()
    for r in (same, small):
        assert all(torch.equal(a, b) for a, b in zip(plain, r))
    # (x is a leaf: kept as it is; the activation's output is kept by its sign)
    assert all(torch.equal(a, b) for a, b in zip(plain, kept))
    with ops.activation_checkpoints8(least=64):
        y = ops.conv2d(x * 1.0, w)
    gw, = torch.autograd.grad(y, w, gy)
    flat = K.plain_codes((x * 1.0).detach().cpu().reshape(1, -1))[2].view(2, 8, -1)
    g = gy.cpu().double().view(2, 16, -1)
    want = sum(g[i] @ flat[i].t() for i in range(2))
    size = sum(g[i].abs() @ flat[i].abs().t() for i in range(2))
    assert ((gw.cpu().double().view(16, 8) - want).abs() <= 2 * K.E32 * 1200 * size).all()
    assert not torch.equal(gw, plain[2])
    # a norm's statistics are no activations: its gradients at a leaf are the same inside
    x8 = K.seeded((4, 16, 6, 5), 6).to(device).contiguous(memory_format=torch.channels_last).requires_grad_()
    for keep in (False, True):
        both = []
        for on in (False, True):
            with ops.activation_checkpoints8(least=40, enabled=on):
                y = ops.group_norm_act(x8, 8, b, b, activation="silu", checkpoint=keep)
            both.append(torch.autograd.grad(y, [x8, b], torch.cos(y.detach())))
        assert all(torch.equal(a, b) for a, b in zip(*both))
    # channels-last, strided and odd-sized saved tensors come back in their order
    for t in (x.detach().movedim(1, -1), x.detach()[:, :, 1:, 1:], x.detach()[:, :3].contiguous()):
        with ops.activation_checkpoints8(least=64):
            a = (t * 1.0).requires_grad_()
            v = (a * 1.0) ** 2
        ga, = torch.autograd.grad(v.sum(), a)
        assert ga.shape == t.shape and ((ga - 2 * t).abs() <= t.abs().max() * 2.0 ** -5).all()


def check_parts(device):
    """each subset of the inputs that can require a gradient gets the same gradients bit for bit; a broadcast gradient, no autograd,
    3 and 5 dimensions, the module"""
    for keep in (False, True):
        for space in ((3, 4), (40, 50)):
            x = K.seeded((3, 24) + space, 1).to(device).contiguous(memory_format=torch.channels_last)
            w, b = K.seeded((24,), 2).to(device), K.seeded((24,), 3).to(device)
            gy = K.seeded((3, 24) + space, 4).to(device)

            def grads(on, gy=gy):
                leaves = [t.clone().requires_grad_(o) for t, o in zip((x, w, b), on)]
                y = ops.group_norm_act(leaves[0], 4, *leaves[1:], activation="silu", checkpoint=keep)
                got = iter(torch.autograd.grad(y, [t for t in leaves if t.requires_grad], gy))
                return [y.detach()] + [next(got) if o else None for o in on]
            whole = grads((True, True, True))
            for on in ((True, False, False), (False, True, False), (False, False, True), (False, True, True), (True, False, True)):
                for got, want in zip(grads(on), whole):
                    assert got is None or torch.equal(got, want), on
            one = torch.ones((), device=device)
            assert all(torch.equal(a, c) for a, c in zip(grads((True,) * 3, one.expand(gy.shape)), grads((True,) * 3, one.expand(gy.shape).clone())))
            with torch.no_grad():
                assert torch.equal(ops.group_norm_act(x, 4, w, b, activation="silu", checkpoint=keep), whole[0])
    flat = ops.group_norm_act(x.flatten(2), 4, w, b)
    assert torch.equal(flat, ops.group_norm_act(x, 4, w, b).flatten(2))
    assert torch.equal(ops.group_norm_act(x.unsqueeze(2), 4, w, b), ops.group_norm_act(x, 4, w, b).unsqueeze(2))
    m, other = ops.GroupNormAct(4, 24, activation="silu").to(device), ops.GroupNormAct(4, 24, activation="silu", checkpoint=True).to(device)
    with torch.no_grad():
        m.weight.copy_(w)
        m.bias.copy_(b)
    assert sorted(m.state_dict()) == ["bias", "weight"]
    other.load_state_dict(m.state_dict())
    assert torch.equal(m(x), other(x)) and torch.equal(m(x), ops.group_norm_act(x, 4, w, b, activation="silu"))


def check_context_twice_differentiated(device):
    """a gradient penalty inside the context: what is saved twice is unpacked with its place in the graph.  Each of the two tensors
    that are kept here is off by 2^-7 of a block's largest value, at most sqrt(32) of the block's root mean square: 2^-3 together"""
    x = K.seeded((2, 8, 16, 16), 1).to(device).requires_grad_()
    w = torch.nn.Parameter(K.seeded((16, 8, 3, 3), 2).to(device))
    b = torch.nn.Parameter(K.seeded((16,), 3).to(device))
    got = []
    for on in (False, True):
        with ops.activation_checkpoints8(least=64, enabled=on):
            y = ops.fused_leaky_relu(ops.conv2d(x, w, padding=1), b)
            g, = torch.autograd.grad((y * torch.cos(y.detach())).sum(), x, create_graph=True)
            penalty = (g * g).sum()
        got.append(torch.autograd.grad(penalty, w)[0].double())
    off = (got[1] - got[0]).norm() / got[0].norm()
    assert 0 < off <= 2 ** -3


@pytest.mark.parametrize("tile", [64, 128, 256])
@pytest.mark.parametrize("dtype", TYPES)
def test_wgrad_every_tile_emulated(emu_lib, dtype, tile, monkeypatch):
    """the tile heights that small sizes do not reach by themselves (the knob exists in tuning builds only)"""
    monkeypatch.setenv("SAE_WG_TILE", str(tile))
    with backend(emu_lib):
        for shape in ((70, 130, 300), (33, 40, 7), (300, 64, 129), (3, 40, 70), (4, 33, 65)):
            K.check_wgrad("cpu", K.TYPES[dtype], shape)


CHECKS = [check_memory_orders, check_empty, check_not_finite, check_linear8, check_run_together, check_context, check_parts, check_context_twice_differentiated]


@pytest.mark.parametrize("check", CHECKS, ids=lambda f: f.__name__[6:])
def test_in_use_emulated(emu_lib, check):
    with backend(emu_lib):
        check("cpu")


# ---- the built library --------------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_gpu_checkpoint8(dtype):
    K.check_checkpoint8("cuda:0", K.TYPES[dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("shape", K.NORM_SHAPES, ids=norm_id)
@pytest.mark.parametrize("dtype", TYPES)
def test_gpu_norm(dtype, shape):
    for i, act in enumerate(ACTS):
        K.check_norm("cuda:0", K.TYPES[dtype], shape, act, checkpoint=False, affine=i != 0)
        K.check_norm("cuda:0", K.TYPES[dtype], shape, act, checkpoint=True, affine=i != 1)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", K.WGRAD_SHAPES, ids=lambda s: "r%d_c%d_o%d" % s)
@pytest.mark.parametrize("dtype", TYPES)
def test_gpu_wgrad(dtype, shape):
    K.check_wgrad("cuda:0", K.TYPES[dtype], shape)
    K.check_wgrad("cuda:0", K.TYPES[dtype], shape, alpha=-0.37, bias=False)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2000, 640, 1100), (4100, 1030, 2048), (1025, 2048, 513), (20000, 256, 250), (3, 2048, 16384), (4, 2048, 16384)], ids=lambda s: "r%d_c%d_o%d" % s)
@pytest.mark.parametrize("dtype", TYPES)
def test_gpu_wgrad_large(dtype, shape):
    """sizes that fill the chip: the tall tiles, slices for every XCD"""
    K.check_wgrad_on_device("cuda:0", K.TYPES[dtype], shape)


@pytest.mark.gpu
@pytest.mark.parametrize("check", CHECKS, ids=lambda f: f.__name__[6:])
def test_gpu_in_use(check):
    check("cuda:0")


def _room(gib):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < gib * 2 ** 30:
        pytest.skip("needs %d GiB of device memory" % gib)


@pytest.mark.gpu
def test_gpu_checkpoint8_past_32_bits():
    """more than 2^31 values: the rows behind are those of a checkpoint of themselves"""
    _room(32)
    x = torch.empty(2 ** 21 + 5, 1030, dtype=torch.bfloat16, device="cuda").normal_()
    kept = ops.checkpoint8(x)
    back = kept.dequantize()
    for part in (slice(0, 9), slice(2 ** 31 // 1056 - 4, 2 ** 31 // 1056 + 4), slice(2 ** 31 // 1030 - 4, 2 ** 31 // 1030 + 4), slice(2 ** 21 - 6, None)):
        own = ops.checkpoint8(x[part])
        assert torch.equal(kept.codes[part], own.codes) and torch.equal(kept.scales[:, part], own.scales)
        assert torch.equal(back[part], own.dequantize())


@pytest.mark.gpu
def test_gpu_norm_past_32_bits():
    """one sample of more than 2^31 values, kept in 8 bits: positions at both ends against the formulas"""
    _room(64)
    l, c, groups = 2 ** 25 + 7, 64, 8
    x = torch.empty(1, l, c, dtype=torch.bfloat16, device="cuda").normal_(0.5, 1.0).movedim(-1, 1).requires_grad_()
    gy = torch.empty(1, l, c, dtype=torch.bfloat16, device="cuda").normal_(0.1, 0.1).movedim(-1, 1)
    w = K.seeded((c,), 1).cuda().requires_grad_()
    y = ops.group_norm_act(x, groups, w, None, activation="silu", checkpoint=True)
    gx, gw = torch.autograd.grad(y, [x, w], gy)
    kept = ops.checkpoint8(x.detach().movedim(1, -1)).dequantize()[0]
    xs, gs, w64 = x.detach()[0].t(), gy[0].t(), w.detach().double()
    step = 2 ** 21
    s1 = sum(xs[i:i + step].double().view(-1, groups, 8).sum((0, 2)) for i in range(0, l, step))
    mean = (s1 / (8 * l)).repeat_interleave(8)
    s2 = sum(((xs[i:i + step].double() - mean) ** 2).view(-1, groups, 8).sum((0, 2)) for i in range(0, l, step))
    rstd = ((s2 / (8 * l)) + 1e-5).rsqrt().repeat_interleave(8)

    def dz_of(part):
        xh = (kept[part].double() - mean) * rstd
        s = torch.sigmoid(xh * w64)
        return gs[part].double() * s * (1 + xh * w64 * (1 - s)), xh
    sums = torch.zeros(4, c, dtype=torch.float64, device="cuda")              # of w dz, w dz xh, dz xh and |dz xh| + |dz|
    for i in range(0, l, step):
        dz, xh = dz_of(slice(i, i + step))
        sums += torch.stack([(w64 * dz).sum(0), (w64 * dz * xh).sum(0), (dz * xh).sum(0), (dz * xh).abs().sum(0) + dz.abs().sum(0)])
    m1, m2 = (t.view(groups, 8).sum(1).repeat_interleave(8) / (8 * l) for t in sums[:2])
    # a thread adds at most 1024 rows; what is in front of the sums is off by 32 roundings of values of at most 1 + |z| at most
    count, u = 1024, K.half_step(torch.bfloat16)
    assert ((gw.double() - sums[2]).abs() <= (count + 32 * 8) * K.E32 * sums[3]).all()
    for part in (slice(0, 500), slice(l - 500, l)):
        z = (xs[part].double() - mean) * rstd * w64
        want = z * torch.sigmoid(z)
        assert ((y.detach()[0].t()[part].double() - want).abs() <= u * want.abs() + 32 * K.E32 * (1 + z.abs()) ** 2).all()
        dz, xh = dz_of(part)
        want = rstd * (w64 * dz - m1 - xh * m2)
        size = rstd * (1 + xh.abs()) * ((w64 * dz).abs() + 1) * (1 + (xh * w64).abs())
        assert ((gx[0].t()[part].double() - want).abs() <= u * want.abs() + (32 + count) * K.E32 * size).all()


@pytest.mark.gpu
def test_gpu_wgrad_past_32_bits():
    """more than 2^31 rows, zeros but for both ends and the middle"""
    _room(96)
    rows, n = 2 ** 31 + 101, 300
    gy = torch.zeros(rows, 1, dtype=torch.float16, device="cuda")
    codes = torch.zeros(rows, 32, dtype=torch.int8, device="cuda")
    scales = torch.full((1, rows), 127, dtype=torch.uint8, device="cuda")
    want = torch.zeros(2, 8, dtype=torch.float64, device="cuda")
    for i, at in enumerate((0, 2 ** 30 + 77, rows - n)):
        x, g = K.seeded((n, 8), i, torch.float16).cuda(), K.seeded((n, 1), 5 + i, torch.float16).cuda()
        own = ops.checkpoint8(x)
        codes[at:at + n], scales[:, at:at + n], gy[at:at + n] = own.codes, own.scales, g
        v = g.double() * own.dequantize().double()
        want += torch.stack([v.sum(0), v.abs().sum(0)])
    gw, gb = ops.linear_weight_grad8(gy, ops.Checkpoint8(codes, scales, 8, torch.float16))
    u = K.half_step(torch.float16)
    assert ((gw[0].double() - want[0]).abs() <= 2 * K.E32 * (3 * n + 32) * want[1] * (1 + u) + u * want[0].abs()).all()
    assert abs(float(gb) - float(gy.double().sum())) <= 2 * K.E32 * (3 * n + 32) * float(gy.abs().double().sum()) * (1 + u) + u * abs(float(gy.double().sum()))


@pytest.mark.gpu
def test_gpu_context_captured():
    """the context inside a captured step: replays with new inputs against the eager step"""
    norm = ops.GroupNormAct(4, 32, activation="silu").cuda()
    w = torch.nn.Parameter(K.seeded((24, 32), 1).cuda())

    def step(x):
        with ops.activation_checkpoints8(least=256):
            y = norm(x * 1.5)
            z = ops.linear8(y.movedim(1, -1), w)
        return torch.autograd.grad(z, [norm.weight, norm.bias, w], 2 * z.detach())
    make = lambda seed: K.seeded((2, 32, 9, 7), seed).cuda().contiguous(memory_format=torch.channels_last)
    x = make(5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x)
    for seed in (6, 7, 8):
        x.copy_(make(seed))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, step(make(seed)))), seed


@pytest.mark.gpu
def test_gpu_two_graphs():
    """two captured steps, replayed in turn and on another stream: each keeps its own workspaces and results"""
    cases = [_step_inputs(30), _step_inputs(40, torch.bfloat16)]
    graphs, outs = [], []
    for c in cases:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _step(*c)
        torch.cuda.current_stream().wait_stream(side)
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(_step(*c))
    want = [_step(*c) for c in cases]
    other = torch.cuda.Stream()
    for turn in range(4):
        for t in outs[0] + outs[1]:
            t.detach().zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(other if turn % 2 else torch.cuda.current_stream()):
            graphs[0].replay()
            graphs[1].replay()
        torch.cuda.synchronize()
        for got, ref in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(got, ref)), turn
        _step(*cases[turn % 2])                                               # eager work in between
        torch.cuda.synchronize()


def _step(x, w, b, gy, wl, gz):
    y = ops.group_norm_act(x, 8, w, b, activation="silu", checkpoint=True)
    g1 = torch.autograd.grad(y, [x, w, b], gy)
    kept = ops.checkpoint8(y.detach().movedim(1, -1))
    g2 = ops.linear_weight_grad8(gz, kept)
    return (y.detach(), kept.dequantize()) + g1 + g2


def _step_inputs(seed, dtype=torch.float32):
    x = K.seeded((2, 33, 17, 64), seed, dtype).cuda().movedim(-1, 1).requires_grad_()
    w, b = K.seeded((64,), seed + 1).cuda().requires_grad_(), K.seeded((64,), seed + 2).cuda().requires_grad_()
    return [x, w, b, K.seeded((2, 33, 17, 64), seed + 3, dtype).cuda().movedim(-1, 1), None, K.seeded((2, 33, 17, 72), seed + 4, dtype).cuda()]


@pytest.mark.gpu
def test_gpu_captured():
    """forward, backward and the weight gradient in one captured graph: replays with new inputs against the eager step, with eager
    work and synchronisations in between"""
    static = _step_inputs(100)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(*static)
    for seed in (200, 300, 400, 500):
        new = _step_inputs(seed)
        with torch.no_grad():
            for s, t in zip(static, new):
                if s is not None:
                    s.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = _step(*new)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), seed


@pytest.mark.gpu
def test_gpu_two_streams_and_repeats():
    """the same step on two streams at once, and again: every result the same bit for bit"""
    cases = [_step_inputs(10), _step_inputs(20, torch.bfloat16)]
    want = [_step(*c) for c in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(_step(*c))
        torch.cuda.synchronize()
        for g, t in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(g, t))
