"""Group normalisation with its activation, channels last (csrc/group_norm.hip).  The reference's networks have no normalisation
with statistics; this stands beside ``fused_leaky_relu`` and ``plane_affine`` for networks that do."""
import torch
from torch import nn
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from .. import hip_lib
from .checkpoint8 import Checkpoint8, empty_checkpoint8

ACTIVATIONS = {"none": 0, "lrelu": 1, "silu": 2}


class GroupNormActFunction(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act, slope, scale, train, keep):
        lib = hip_lib.get()
        x = hip_lib.dense(x.movedim(1, -1))                 # [n, ..., c]; no copy for a channels-last tensor
        weight = None if weight is None else weight.contiguous()
        bias = None if bias is None else bias.contiguous()
        lib.check_channels_last(x)
        n, c = x.shape[0], x.shape[-1]
        l = x.shape[1:-1].numel()
        y = torch.empty_like(x)
        stats = torch.empty(2, n, groups, dtype=torch.float32, device=x.device)
        kept = empty_checkpoint8(x) if keep else None
        dt = hip_lib.element_types()[x.dtype]
        n_ws = lib.query("group_norm_act_workspace", n, l, c, groups, dt, 0)
        ws = torch.empty(max(n_ws, 1), dtype=torch.uint8, device=x.device)
        with lib.device_of(x):
            lib.call("group_norm_act", x.data_ptr(), hip_lib.ptr(weight), hip_lib.ptr(bias), y.data_ptr(), stats[0].data_ptr(),
                     stats[1].data_ptr(), kept.codes.data_ptr() if keep else None, kept.scales.data_ptr() if keep else None, n, l, c,
                     groups, eps, act, slope, scale, dt, ws.data_ptr(), n_ws, lib.stream(x))
        if train:
            ctx.save_for_backward(weight, bias, stats, *((kept.codes, kept.scales) if keep else (x,)))
            ctx.cfg = (n, l, c, groups, act, slope, scale, dt)
        return y.movedim(-1, 1)

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        weight, bias, stats, *rest = ctx.saved_tensors
        n, l, c, groups, act, slope, scale, dt = ctx.cfg
        lib = hip_lib.get()
        gy = hip_lib.dense(gy.movedim(1, -1))
        lib.check_channels_last(gy)
        x, codes, scales = (None, *rest) if len(rest) == 2 else (rest[0], None, None)
        gx = torch.empty_like(gy) if ctx.needs_input_grad[0] else None
        gw = torch.empty_like(weight) if ctx.needs_input_grad[1] else None
        gb = torch.empty_like(bias) if ctx.needs_input_grad[2] else None
        n_ws = lib.query("group_norm_act_workspace", n, l, c, groups, dt, 1)
        ws = torch.empty(max(n_ws, 1), dtype=torch.uint8, device=gy.device)
        with lib.device_of(gy):
            lib.call("group_norm_act_bwd", gy.data_ptr(), hip_lib.ptr(x), hip_lib.ptr(codes), hip_lib.ptr(scales),
                     stats[0].data_ptr(), stats[1].data_ptr(), hip_lib.ptr(weight), hip_lib.ptr(bias), hip_lib.ptr(gx),
                     hip_lib.ptr(gw), hip_lib.ptr(gb), n, l, c, groups, act, slope, scale, dt, ws.data_ptr(), n_ws, lib.stream(gy))
        return None if gx is None else gx.movedim(-1, 1), gw, gb, None, None, None, None, None, None, None


def group_norm_act(input, num_groups, weight=None, bias=None, eps=1e-5, activation="lrelu", negative_slope=0.2, scale=None,
                   checkpoint=False):
    """scale * act((x - mean) * rstd * weight + bias) of x [N, C, ...], mean and variance over each sample's C / num_groups
    channels and all of its positions.

    activation: "lrelu" (negative_slope; scale 2 ** 0.5 unless given, as ``fused_leaky_relu``), "silu" or "none" (scale 1 unless
    given).  x: float32, bfloat16 or float16, channels last in memory (any other order is copied into it); the result is channels
    last.  weight, bias: float32 [C] or None.  checkpoint: the backward pass works from the 8-bit checkpoint of x that the forward
    writes beside y, instead of from x (``checkpoint8``); y is the same, the gradients are those at the values it stands for.
    Differentiable once."""
    if activation not in ACTIVATIONS:
        raise hip_lib.SaeError("group_norm_act: activation must be one of %s, got %r" % (sorted(ACTIVATIONS), activation))
    if input.dim() < 2 or input.shape[1] < 1 or num_groups < 1 or input.shape[1] % num_groups:
        raise hip_lib.SaeError("group_norm_act: x must be [N, C, ...] with C a multiple of num_groups = %d, got %s"
                               % (num_groups, tuple(input.shape)))
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and (t.dtype != torch.float32 or tuple(t.shape) != (input.shape[1],) or t.device != input.device):
            raise hip_lib.SaeError("group_norm_act: %s must be float32 [%d] on %s, got %s %s on %s"
                                   % (name, input.shape[1], input.device, t.dtype, tuple(t.shape), t.device))
    if not eps >= 0:
        raise hip_lib.SaeError("group_norm_act: eps must not be negative, got %r" % (eps,))
    if scale is None:
        scale = 2 ** 0.5 if activation == "lrelu" else 1.0
    train = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (input, weight, bias))
    return GroupNormActFunction.apply(input, weight, bias, int(num_groups), float(eps), ACTIVATIONS[activation],
                                      float(negative_slope), float(scale), train, bool(checkpoint) and train)


class GroupNormAct(nn.Module):
    """``group_norm_act`` with its parameters (weight one, bias zero)."""

    def __init__(self, num_groups, channel, eps=1e-5, activation="lrelu", negative_slope=0.2, scale=None, checkpoint=False):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(channel))
        self.bias = nn.Parameter(torch.zeros(channel))
        self.num_groups, self.eps, self.activation = num_groups, eps, activation
        self.negative_slope, self.scale, self.checkpoint = negative_slope, scale, checkpoint

    def forward(self, input):
        return group_norm_act(input, self.num_groups, self.weight, self.bias, self.eps, self.activation, self.negative_slope,
                              self.scale, self.checkpoint)
