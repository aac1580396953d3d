"""Group normalisation with its activation, channels last (csrc/group_norm.hip).  The reference's networks have no normalisation
with statistics; this stands beside ``fused_leaky_relu`` and ``plane_affine`` for networks that do."""
import torch
from torch import nn
from torch.autograd import Function, forward_ad
from torch.autograd.function import once_differentiable

from .. import hip_lib
from .checkpoint8 import BLOCK

ACTIVATIONS = {"none": 0, "lrelu": 1, "silu": 2}


def _last(x):
    """(dense memory [n, ..., c] of x [n, c, ...], n, positions, c); no copy for a channels-last tensor."""
    shape = x.shape
    if len(shape) == 4 and x.is_contiguous(memory_format=torch.channels_last) and x.data_ptr() % 16 == 0 and not x.is_neg():
        return x, shape[0], shape[2] * shape[3], shape[1]
    return hip_lib.dense(x.movedim(1, -1)).movedim(-1, 1), shape[0], shape[2:].numel(), shape[1]


def _forward(lib, x, weight, bias, groups, eps, act, slope, scale, keep):
    """(y, x as it is read, stats [2, n, groups], codes, scales)"""
    code = lib.check_channels_last(x)
    x, n, l, c = _last(x)
    y = torch.empty_like(x)                                # (channels last, as x is)
    stats = x.new_empty((2, n, groups), dtype=torch.float32)
    codes = scales = None
    if keep:
        blocks = -(-c // BLOCK)
        codes, scales = x.new_empty((n * l, BLOCK * blocks), dtype=torch.int8), x.new_empty((blocks, n * l), dtype=torch.uint8)
    n_ws = lib.query("group_norm_act_workspace", n, l, c, groups, code, 0)
    ws = x.new_empty((n_ws,), dtype=torch.uint8) if n_ws else None
    ptr = hip_lib.ptr
    mean = stats.data_ptr()
    lib.call_on(x, "group_norm_act", x.data_ptr(), ptr(weight), ptr(bias), y.data_ptr(), mean, mean + 4 * n * groups, ptr(codes),
                ptr(scales), n, l, c, groups, eps, act, slope, scale, code, ptr(ws), n_ws)
    return y, x, stats, codes, scales


class GroupNormActFunction(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act, slope, scale, keep):
        y, x, stats, codes, scales = _forward(hip_lib.get(), x, weight, bias, groups, eps, act, slope, scale, keep)
        if keep:
            ctx.save_for_backward(weight, bias, None, codes, scales)
        else:
            ctx.save_for_backward(weight, bias, x, None, None)
        ctx.stats = stats                                  # (no activation: saved-tensor hooks that round those leave it alone)
        ctx.cfg = (groups, act, slope, scale)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        weight, bias, x, codes, scales = ctx.saved_tensors
        groups, act, slope, scale = ctx.cfg
        lib = hip_lib.get()
        code = lib.check_channels_last(gy)
        if x is not None:
            x = _last(x)[0]
        gy, n, l, c = _last(gy)
        need = ctx.needs_input_grad
        gx = torch.empty_like(gy) if need[0] else None
        gw = torch.empty_like(weight) if need[1] else None
        gb = torch.empty_like(bias) if need[2] else None
        n_ws = lib.query("group_norm_act_workspace", n, l, c, groups, code, 1)
        ws = gy.new_empty((n_ws,), dtype=torch.uint8) if n_ws else None
        ptr = hip_lib.ptr
        mean = ctx.stats.data_ptr()
        lib.call_on(gy, "group_norm_act_bwd", gy.data_ptr(), ptr(x), ptr(codes), ptr(scales), mean, mean + 4 * n * groups,
                    ptr(weight), ptr(bias), ptr(gx), ptr(gw), ptr(gb), n, l, c, groups, act, slope, scale, code, ptr(ws), n_ws)
        return gx, gw, gb, None, None, None, None, None, None


def group_norm_act(input, num_groups, weight=None, bias=None, eps=1e-5, activation="lrelu", negative_slope=0.2, scale=None,
                   checkpoint=False):
    """scale * act((x - mean) * rstd * weight + bias) of x [N, C, ...], mean and variance over each sample's C / num_groups
    channels and all of its positions.  Up to 65535 samples and groups and 2 ** 20 channels; what exceeds them is refused.

    activation: "lrelu" (negative_slope; scale 2 ** 0.5 unless given, as ``fused_leaky_relu``), "silu" or "none" (scale 1 unless
    given).  x: float32, bfloat16 or float16, channels last in memory (any other order is copied into it); the result is channels
    last.  weight, bias: float32 [C] or None.  checkpoint: the backward pass works from the 8-bit checkpoint of x that the forward
    writes beside y, instead of from x (``checkpoint8``); y is the same but for the rounding of the statistics (rows are dealt out
    to threads in whole blocks of 32 channels then), the gradients are those at the values it stands for.
    Differentiable once, in reverse mode."""
    if activation not in ACTIVATIONS:
        raise hip_lib.SaeError("group_norm_act: activation must be one of %s, got %r" % (sorted(ACTIVATIONS), activation))
    if input.dim() < 2 or input.shape[1] < 1 or num_groups < 1 or input.shape[1] % num_groups:
        raise hip_lib.SaeError("group_norm_act: x must be [N, C, ...] with C a multiple of num_groups = %d, got %s"
                               % (num_groups, tuple(input.shape)))
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and (t.dtype != torch.float32 or t.shape != input.shape[1:2] or t.device != input.device):
            raise hip_lib.SaeError("group_norm_act: %s must be float32 [%d] on %s, got %s %s on %s"
                                   % (name, input.shape[1], input.device, t.dtype, tuple(t.shape), t.device))
    if not eps >= 0:
        raise hip_lib.SaeError("group_norm_act: eps must not be negative, got %r" % (eps,))
    if scale is None:
        scale = 2 ** 0.5 if activation == "lrelu" else 1.0
    weight = weight if weight is None or weight.is_contiguous() else weight.contiguous()
    bias = bias if bias is None or bias.is_contiguous() else bias.contiguous()
    # (a forward-mode level: by the Function, which refuses a tangent)
    if forward_ad._current_level >= 0 or torch.is_grad_enabled() and (
            input.requires_grad or (weight is not None and weight.requires_grad) or (bias is not None and bias.requires_grad)):
        return GroupNormActFunction.apply(input, weight, bias, num_groups, eps, ACTIVATIONS[activation], negative_slope, scale,
                                          bool(checkpoint))
    return _forward(hip_lib.get(), input, weight, bias, num_groups, eps, ACTIVATIONS[activation], negative_slope, scale, False)[0]


class GroupNormAct(nn.Module):
    """``group_norm_act`` with its parameters (weight one, bias zero), which stay float32 for every type of input: convert the
    activations, not the module."""

    def __init__(self, num_groups, channel, eps=1e-5, activation="lrelu", negative_slope=0.2, scale=None, checkpoint=False):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(channel))
        self.bias = nn.Parameter(torch.zeros(channel))
        self.num_groups, self.eps, self.activation = num_groups, eps, activation
        self.negative_slope, self.scale, self.checkpoint = negative_slope, scale, checkpoint

    def forward(self, input):
        return group_norm_act(input, self.num_groups, self.weight, self.bias, self.eps, self.activation, self.negative_slope,
                              self.scale, self.checkpoint)
