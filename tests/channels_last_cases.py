"""Inputs, 64-bit plain forms and error bounds of the channels-last operators (group_norm_act, checkpoint8, linear_weight_grad8),
shared by the CPU tests (the kernel sources on the emulator) and the GPU tests (the built library)."""
import numpy as np
import torch

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
LEAST = {torch.float32: -126, torch.bfloat16: -126, torch.float16: -24}
MOST = {torch.float32: 121, torch.bfloat16: 121, torch.float16: 9}
E32 = 2.0 ** -24                                                       # half a step of fp32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def seeded(shape, seed, dtype=torch.float32, mean=0.0, size=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * size + mean).to(dtype)


# ---- 8-bit checkpoints --------------------------------------------------------------------------------------------------------

def plain_codes(x):
    """(codes [rows, 32 blocks] int8, scales [blocks, rows] uint8, values [rows, c] float64) of x [rows, c], block by block"""
    rows, c = x.shape
    blocks = -(-c // 32)
    v = x.double().numpy()
    codes = np.zeros((rows, 32 * blocks), np.int8)
    scales = np.zeros((blocks, rows), np.uint8)
    values = np.zeros((rows, c))
    for r in range(rows):
        for b in range(blocks):
            part = v[r, 32 * b:32 * b + 32]
            if not np.isfinite(part).all():
                scales[b, r] = 255
                values[r, 32 * b:32 * b + 32] = np.nan
                continue
            top, k = np.abs(part).max(), LEAST[x.dtype]
            while k < MOST[x.dtype] and top > np.ldexp(127.5, k):
                k += 1
            q = np.clip(np.rint(np.ldexp(part, -k)), -127, 127)
            q = np.where((q == 0) & (part != 0), np.sign(part), q)
            scales[b, r] = k + 127
            codes[r, 32 * b:32 * b + len(part)] = q
            values[r, 32 * b:32 * b + 32] = np.ldexp(q, k)
    return torch.from_numpy(codes), torch.from_numpy(scales), torch.from_numpy(values)


def awkward(dtype):
    """Rows of 70 values (two whole blocks and a short one) with what a block can meet"""
    top = torch.finfo(dtype).max
    tiny = 2.0 ** -24 if dtype == torch.float16 else 2.0 ** -133 if dtype == torch.bfloat16 else 2.0 ** -149
    x = torch.zeros(14, 70, dtype=torch.float64)
    base = seeded((14, 70), 5).double()
    x[1] = base[1]
    x[2] = base[2] * 1e-4
    x[3] = top * torch.linspace(-1, 1, 70)
    x[4] = tiny * torch.arange(70)
    x[5] = base[5]
    x[5, 3], x[5, 40] = float("nan"), float("inf")
    x[6] = base[6]
    x[6, 69] = float("-inf")
    x[7] = torch.arange(70) - 35.0                       # whole steps
    x[8] = (torch.arange(70) - 35.0) * 0.5               # ties
    x[8, 0], x[8, 32], x[8, 64] = 127.0, -127.0, 100.0
    x[9] = base[9]
    x[9, 0], x[9, 33] = 127.5, 127.5 * 2 ** 3            # the border of a step
    x[10] = base[10] * 1e-3
    x[10, 7], x[10, 65] = -1e4, 3e4                      # one value far above the others
    x[11, 31] = 1.0                                      # a block of zeros but one, blocks of zeros
    x[12] = -base[12].abs()
    x[13] = 2.0 ** -14 * (1 + torch.arange(70) / 70)
    return x.to(dtype)


PACK_SHAPES = [(1, 1), (3, 31), (5, 32), (2, 33), (7, 72), (4, 515), (70, 64), (1, 4096), (300, 8)]


def check_checkpoint8(device, dtype):
    from swapping_autoencoder_pytorch_amd.stylegan2_op import checkpoint8
    for x in [awkward(dtype)] + [seeded(s, 3 + i, dtype, 0.3, 2.0) for i, s in enumerate(PACK_SHAPES)]:
        kept = checkpoint8(x.to(device))
        codes, scales, values = plain_codes(x)
        assert torch.equal(kept.codes.cpu(), codes), tuple(x.shape)
        assert torch.equal(kept.scales.cpu(), scales), tuple(x.shape)
        back = kept.dequantize()
        assert back.dtype == dtype and back.shape == x.shape and back.is_contiguous()
        assert torch.equal(torch.nan_to_num(back.cpu().double(), nan=-1e300), torch.nan_to_num(values, nan=-1e300)), tuple(x.shape)
        # what the format promises: sign exact, off by half a step at most (one step where that would make a zero, or next to the
        # type's largest number)
        fine = torch.isfinite(values)
        step = torch.from_numpy(np.ldexp(1.0, scales.numpy().astype(int) - 127)).t().repeat_interleave(32, 1)[:, :x.shape[1]]
        off = (back.cpu().double() - x.double()).abs()
        assert torch.equal(torch.sign(back.cpu().double())[fine], torch.sign(x.double())[fine])
        assert (off[fine] <= torch.where((x.double().abs() < step / 2) | (x.double().abs() > 127.5 * step), step, step / 2)[fine]).all()


# ---- group normalisation ------------------------------------------------------------------------------------------------------

# n, positions, channels, groups: vectors of whole groups, groups that cut a vector, odd channels (one channel a lane), rows wider
# than a work-group, single positions and channels, one group for all, several chunks of rows
NORM_SHAPES = [(2, (5, 7), 32, 8), (3, (4, 3), 100, 20), (1, (1, 1), 64, 16), (2, (3, 5), 72, 8), (1, (2,), 5, 5), (2, (9,), 1, 1),
               (1, (3, 2), 1030, 2), (1, (2, 2), 2048, 32), (2, (23, 27), 16, 4), (3, (), 48, 6), (2, (17, 3), 40, 1),
               (1, (70, 5), 24, 3)]


def act64(z, act, slope):
    if act == "lrelu":
        return torch.where(z > 0, z, slope * z)
    return z / (1 + torch.exp(-z)) if act == "silu" else z


def act_slope64(z, act, slope):
    if act == "lrelu":
        return torch.where(z > 0, torch.ones_like(z), torch.full_like(z, slope))
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def norm64(x, kept, gy, groups, w, b, eps, act, slope, scale):
    """y, gx, gw, gb in 64 bits by the formulas, with what the bounds need; x, gy [n, c, ...] of the inputs' own values; kept: what
    the backward pass works from"""
    n, c = x.shape[:2]
    x, kept, gy = (t.double().reshape(n, groups, c // groups, -1) for t in (x, kept, gy))
    w64 = (torch.ones(c) if w is None else w).double().view(1, groups, -1, 1)
    b64 = (torch.zeros(c) if b is None else b).double().view(1, groups, -1, 1)
    mean = x.mean((2, 3), keepdim=True)
    rstd = (((x - mean) ** 2).mean((2, 3), keepdim=True) + eps) ** -0.5
    z = (x - mean) * rstd * w64 + b64
    y = scale * act64(z, act, slope)
    xh = (kept - mean) * rstd
    zk = xh * w64 + b64
    dz = gy * scale * act_slope64(zk, act, slope)
    wd = w64 * dz
    m1, m2 = wd.mean((2, 3), keepdim=True), (wd * xh).mean((2, 3), keepdim=True)
    gx = rstd * (wd - m1 - xh * m2)
    # error of z: roundings of mean, x - mean, rstd, rstd * w, the sum: each half a step of a number of this size
    big = w64.abs() * (xh.abs() + mean.abs() * rstd) + b64.abs()
    big_y = w64.abs() * ((x - mean).abs() * rstd + mean.abs() * rstd) + b64.abs()
    rows = x.shape[3]
    # y: those eight, and the activation's (exponent's argument and value, sum, reciprocal, product, scale) at (1 + |z|)
    ey = scale * 16 * E32 * big_y * (1 + z.abs()) + half_step_of(y)
    # dz: its own roundings, and what the error of z moves the slope by (at most a half for silu, nothing for the others)
    ed = (gy * scale).abs() * 16 * E32 * (1 + zk.abs() + big)
    ewd = w64.abs() * ed
    # sums: a thread adds at most all rows one after the other, the rest are a few more
    count = rows + 64
    em1 = ewd.mean((2, 3), keepdim=True) + count * E32 * wd.abs().mean((2, 3), keepdim=True)
    exh = 8 * E32 * (xh.abs() + mean.abs() * rstd)
    em2 = (ewd * xh.abs() + wd.abs() * exh).mean((2, 3), keepdim=True) + count * E32 * (wd * xh).abs().mean((2, 3), keepdim=True)
    egx = rstd * (ewd + em1 + exh * m2.abs() + xh.abs() * em2 + 8 * E32 * (wd.abs() + m1.abs() + (xh * m2).abs()))
    egb = (ed + count * E32 * dz.abs()).sum((0, 3))
    egw = (ed * xh.abs() + dz.abs() * exh + count * E32 * (dz * xh).abs()).sum((0, 3))
    kink = zk.abs() <= 16 * E32 * big if act == "lrelu" else torch.zeros_like(zk, dtype=torch.bool)
    return dict(y=y, gx=gx, gw=(dz * xh).sum((0, 3)).view(-1), gb=dz.sum((0, 3)).view(-1), ey=ey, egx=egx, egw=egw.view(-1),
                egb=egb.view(-1), kink=kink, mean=mean, rstd=rstd)


def half_step_of(v):
    return E32 * v.abs()


def check_norm(device, dtype, shape, act, checkpoint, affine=True, mean=0.5, memory="channels_last", slope=0.2, scale=None, seed=0):
    from swapping_autoencoder_pytorch_amd.stylegan2_op import group_norm_act
    n, space, c, groups = shape
    full = (n, c) + tuple(space)
    x = (seeded(full, 10 + seed, mean=mean) * (0.5 + seeded((c,), 11 + seed).abs()).view((1, c) + (1,) * len(space))).to(dtype)
    gy = seeded(full, 12 + seed, dtype, 0.0, 0.1)
    w, b = (1 + 0.3 * seeded((c,), 13 + seed), 0.2 * seeded((c,), 14 + seed)) if affine else (None, None)

    def place(t):
        t = t.to(device)
        if memory == "channels_last":
            return t.movedim(1, -1).contiguous().movedim(-1, 1)
        if memory == "sliced":                      # inside a larger tensor: strided, not aligned
            h = torch.zeros(tuple(s + 1 for s in t.shape), dtype=t.dtype, device=t.device)
            h[tuple(slice(1, None) for _ in t.shape)] = t
            return h[tuple(slice(1, None) for _ in t.shape)]
        return t

    leaves = [place(x).requires_grad_()] + [t.to(device).requires_grad_() for t in (w, b) if t is not None]
    y = group_norm_act(leaves[0], groups, *(leaves[1:] or [None, None]), activation=act, negative_slope=slope, scale=scale,
                       checkpoint=checkpoint)
    assert y.dtype == dtype and tuple(y.shape) == full and y.movedim(1, -1).is_contiguous()
    grads = torch.autograd.grad(y, leaves, place(gy))
    kept = x
    if checkpoint:
        kept = plain_codes(x.movedim(1, -1).reshape(-1, c))[2].view((n,) + tuple(space) + (c,)).movedim(-1, 1)
    scale = (2 ** 0.5 if act == "lrelu" else 1.0) if scale is None else scale
    r = norm64(x, kept, gy, groups, w, b, 1e-5, act, slope, scale)
    u = half_step(dtype)

    def near(got, want, bound, skip=None):
        off = (got.detach().cpu().double().reshape(want.shape) - want).abs()
        over = off - (bound * (1 + u) + u * want.abs() + torch.finfo(dtype).smallest_normal * u)
        if skip is not None:
            over = torch.where(skip, torch.full_like(over, -1.0), over)
        assert not torch.isnan(off).any() and (over <= 0).all(), (shape, act, checkpoint, float(over.max()), float(off.max()))

    near(y, r["y"], r["ey"])
    near(grads[0], r["gx"], r["egx"], r["kink"])
    if affine:
        assert grads[1].dtype == grads[2].dtype == torch.float32
        if not r["kink"].any():
            near(grads[1], r["gw"], r["egw"])
            near(grads[2], r["gb"], r["egb"])


# ---- weight gradient ----------------------------------------------------------------------------------------------------------

# rows, channels of x, channels of gy: single values, odd ones, each tile height, several tiles, several slices with a short end
WGRAD_SHAPES = [(1, 1, 1), (5, 33, 7), (32, 64, 64), (33, 130, 100), (100, 40, 128), (64, 128, 300), (257, 20, 260), (31, 515, 130),
                (700, 96, 12)]


def check_wgrad(device, dtype, shape, alpha=1.0, bias=True):
    from swapping_autoencoder_pytorch_amd.stylegan2_op import checkpoint8, linear_weight_grad8
    rows, c, out = shape
    x, gy = seeded((rows, c), 20, dtype, 0.2), seeded((rows, out), 21, dtype, 0.0, 0.3)
    gw, gb = linear_weight_grad8(gy.to(device), checkpoint8(x.to(device)), bias=bias, alpha=alpha)
    values = plain_codes(x)[2]
    u, g = half_step(dtype), gy.double()
    # products exact; every addition of the fp32 sum off by one step at most (cut or rounded); slices, alpha and the store behind
    want, size = alpha * g.t() @ values, abs(alpha) * g.abs().t() @ values.abs()
    assert gw.dtype == dtype and tuple(gw.shape) == (out, c)
    assert ((gw.cpu().double() - want).abs() <= 2 * E32 * (rows + 32) * size * (1 + u) + u * want.abs() + 1e-30).all(), shape
    if not bias:
        assert gb is None
        return
    assert gb.dtype == dtype and tuple(gb.shape) == (out,)
    assert ((gb.cpu().double() - g.sum(0)).abs() <= 2 * E32 * (rows + 32) * g.abs().sum(0) * (1 + u) + u * g.sum(0).abs() + 1e-30).all()


def check_wgrad_on_device(device, dtype, shape):
    """check_wgrad at sizes where the reference is computed on the device as well (its own float64 products)"""
    from swapping_autoencoder_pytorch_amd.stylegan2_op import checkpoint8, linear_weight_grad8
    rows, c, out = shape
    x, gy = seeded((rows, c), 20, dtype, 0.2).to(device), seeded((rows, out), 21, dtype, 0.0, 0.3).to(device)
    kept = checkpoint8(x)
    gw, gb = linear_weight_grad8(gy, kept)
    v, g, u = kept.dequantize().double(), gy.double().t().contiguous(), half_step(dtype)
    want, size = g @ v, g.abs() @ v.abs()
    assert ((gw.double() - want).abs() <= 2 * E32 * (rows + 32) * size * (1 + u) + u * want.abs()).all()
    want, size = g.sum(1), g.abs().sum(1)
    assert ((gb.double() - want).abs() <= 2 * E32 * (rows + 32) * size * (1 + u) + u * want.abs()).all()
