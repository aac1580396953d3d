"""8-bit activation checkpoints: what a backward pass needs of the forward pass, kept in a quarter (f32) or half (bf16, f16) of
its size, and the operators that read it there (csrc/checkpoint8.hip, csrc/linear_wgrad8.hip).

The format (csrc/elem8.inc): blocks of 32 values along the last dimension with one power-of-two step each and a signed 8-bit code
for each value.  A step is 1 / 127.5 ... 1 / 63.75 of the block's largest value (more where that is next to the smallest step, 2^-126,
or 2^-24 in f16).  Values of at least half a step are off by half a step at most; what is smaller and not zero becomes one step, off
by less than that, so that only a zero becomes zero and sign(x) is exact -- the mask that a leaky ReLU's backward reads.  (Next to
the type's largest number, above 127.5 steps of the largest step, the error is up to one step.)  A block with a NaN or an infinity
comes back as NaN.

  checkpoint8               activation -> Checkpoint8, ``.dequantize()`` gives it back
  linear_weight_grad8       weight and bias gradient of a linear layer from the Checkpoint8 of its input
  linear8                   ``linear`` that keeps its input as a Checkpoint8
  activation_checkpoints8   every node built inside keeps the activations it saves as Checkpoint8s

The reference keeps every activation in fp32 (it never enables AMP)."""
import contextlib
import weakref

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable
from torch.multiprocessing.reductions import StorageWeakRef

from .. import hip_lib
from .conv2d_gemm import _Flags, _gemm

BLOCK = 32


class Checkpoint8:
    """codes int8 [rows, 32 * blocks] (zero behind a row's last value), scales uint8 [blocks, rows] (exponent of the step + 127,
    255: NaN), blocks = ceil(channels / 32); stands for a tensor of ``shape`` (default [rows, channels]) and ``dtype``."""
    __slots__ = ("codes", "scales", "channels", "dtype", "shape")

    def __init__(self, codes, scales, channels, dtype, shape=None):
        blocks = -(-channels // BLOCK)
        if channels < 1 or dtype not in hip_lib.element_types():
            raise hip_lib.SaeError("Checkpoint8: channels >= 1 and float32 / bfloat16 / float16, got %d, %s" % (channels, dtype))
        if codes.dtype != torch.int8 or codes.dim() != 2 or codes.shape[1] != BLOCK * blocks or not codes.is_contiguous():
            raise hip_lib.SaeError("Checkpoint8: codes must be contiguous int8 [rows, %d], got %s %s"
                                   % (BLOCK * blocks, codes.dtype, tuple(codes.shape)))
        if scales.dtype != torch.uint8 or tuple(scales.shape) != (blocks, codes.shape[0]) or not scales.is_contiguous():
            raise hip_lib.SaeError("Checkpoint8: scales must be contiguous uint8 %s, got %s %s"
                                   % ((blocks, codes.shape[0]), scales.dtype, tuple(scales.shape)))
        if codes.device != scales.device:
            raise hip_lib.SaeError("Checkpoint8: codes on %s, scales on %s" % (codes.device, scales.device))
        shape = torch.Size((codes.shape[0], channels) if shape is None else shape)
        if not shape or shape[-1] != channels or shape[:-1].numel() != codes.shape[0]:
            raise hip_lib.SaeError("Checkpoint8: shape %s is not %d rows of %d" % (tuple(shape), codes.shape[0], channels))
        self.codes, self.scales, self.channels, self.dtype, self.shape = hip_lib.dense(codes), scales, channels, dtype, shape

    @classmethod
    def _of(cls, codes, scales, channels, dtype, shape):
        """From parts that are known to fit."""
        self = object.__new__(cls)
        self.codes, self.scales, self.channels, self.dtype, self.shape = codes, scales, channels, dtype, shape
        return self

    @property
    def rows(self):
        return self.codes.shape[0]

    @property
    def nbytes(self):
        return self.codes.numel() + self.scales.numel()

    def dequantize(self):
        """The values the codes stand for, a new contiguous tensor."""
        lib = hip_lib.get()
        x = torch.empty(self.shape, dtype=self.dtype, device=self.codes.device)
        code = lib.check_channels_last(x)
        lib.call_on(x, "checkpoint8_unpack", self.codes.data_ptr(), self.scales.data_ptr(), x.data_ptr(), self.codes.shape[0],
                    self.channels, code)
        return x


def empty_checkpoint8(x):
    """Checkpoint8 of x's type for rows x's leading dimensions, not yet written."""
    shape = x.shape
    channels = shape[-1]
    rows = shape[0] if len(shape) == 2 else shape[:-1].numel()
    blocks = -(-channels // BLOCK)
    return Checkpoint8._of(x.new_empty((rows, BLOCK * blocks), dtype=torch.int8), x.new_empty((blocks, rows), dtype=torch.uint8),
                           channels, x.dtype, shape)


def checkpoint8(x):
    """The 8-bit checkpoint of x [..., channels] (no gradient flows through it).  Blocks run along the last dimension: hand a
    channels-last image over as ``x.movedim(1, -1)``."""
    if x.dim() < 1 or x.shape[-1] < 1:
        raise hip_lib.SaeError("checkpoint8: at least one value in the last dimension, got shape %s" % (tuple(x.shape),))
    lib = hip_lib.get()
    code = lib.check_channels_last(x)
    x = hip_lib.dense(x.detach())
    kept = empty_checkpoint8(x)
    lib.call_on(x, "checkpoint8_pack", x.data_ptr(), kept.codes.data_ptr(), kept.scales.data_ptr(), kept.codes.shape[0],
                kept.channels, code)
    return kept


def linear_weight_grad8(gy, kept, bias=True, alpha=1.0):
    """(gw [out, channels], gb [out] or None) of ``alpha * x @ weight.T + bias`` from gy [..., out] and the Checkpoint8 of x:
    gw = alpha * gy^T x8, gb = the sum of gy's rows (no gradient flows through them).  In gy's type, which has to be the
    checkpoint's; the products are exact and added in fp32 (f32: gy in three bf16 pieces, which hold all of its 24 bits from 2^-110 up
    and are off by less than 2^-132 below)."""
    lib = hip_lib.get()
    shape, codes = gy.shape, kept.codes
    rows, out, c = codes.shape[0], shape[-1] if shape else 0, kept.channels
    if out < 1 or (shape[0] if len(shape) == 2 else shape[:-1].numel()) != rows:
        raise hip_lib.SaeError("linear_weight_grad8: gy %s does not have the checkpoint's %d rows" % (tuple(shape), rows))
    if gy.dtype != kept.dtype or gy.device != codes.device:
        raise hip_lib.SaeError("linear_weight_grad8: gy is %s on %s, the checkpoint %s on %s"
                               % (gy.dtype, gy.device, kept.dtype, codes.device))
    code = lib.check_channels_last(gy)
    gy = hip_lib.dense(gy.detach())
    gw = gy.new_empty((out, c))
    gb = gy.new_empty((out,)) if bias else None
    n_ws = lib.query("linear_wgrad8_workspace", rows, out, c, code)
    ws = gy.new_empty((n_ws,), dtype=torch.float32) if n_ws else None
    lib.call_on(gy, "linear_wgrad8", gy.data_ptr(), codes.data_ptr(), kept.scales.data_ptr(), gw.data_ptr(), hip_lib.ptr(gb), rows,
                out, c, alpha, code, hip_lib.ptr(ws), n_ws)
    return gw, gb


class Linear8(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, alpha, train):
        y = _gemm(x, weight, bias, False, True, alpha)
        if train:
            kept = checkpoint8(x) if weight.requires_grad else None
            ctx.save_for_backward(weight, *((kept.codes, kept.scales) if kept is not None else ()))
            ctx.cfg = (alpha, bias is not None)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        weight, *kept = ctx.saved_tensors
        alpha, has_bias = ctx.cfg
        gy = hip_lib.dense(gy)
        gx = gw = gb = None
        if ctx.needs_input_grad[0]:
            gx = _gemm(gy, weight, None, False, False, alpha)
        if ctx.needs_input_grad[1] and _Flags.weight_grads:
            gw, gb = linear_weight_grad8(gy, Checkpoint8._of(*kept, weight.shape[1], torch.float32, None), has_bias, alpha)
        if ctx.needs_input_grad[2] and gb is None:
            gb = _gemm(gy.new_ones((1, gy.shape[0])), gy, None, False, False, 1.0)[0]     # (a captured step: no sum of torch's)
        return gx, gw, gb, None, None


def linear8(input, weight, bias=None, alpha=1.0):
    """``linear`` (alpha * input @ weight^T + bias, float32) whose backward takes the weight gradient from the 8-bit checkpoint of
    the input; y and the input gradient are ``linear``'s.  Differentiable once."""
    if input.dim() < 1 or weight.dim() != 2:
        raise hip_lib.SaeError("linear8: input [..., in] and weight [out, in], got %s and %s" % (tuple(input.shape), tuple(weight.shape)))
    lead = input.shape[:-1]
    x2 = input.reshape(-1, input.shape[-1])
    train = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (input, weight, bias))
    return Linear8.apply(x2, weight, bias, alpha, train).view(*lead, weight.shape[0])


def _lives_anyway(t):
    """A parameter, trainable or frozen, another leaf that requires a gradient, or a view of one: its memory is not the graph's to
    free, and a data gradient through it would be taken at rounded weights."""
    base = t if t._base is None else t._base
    return isinstance(base, torch.nn.Parameter) or (base.is_leaf and base.requires_grad)


class _Kept:
    """One packed activation: the checkpoint of its memory in order, and the strides it had."""
    __slots__ = ("kept", "size", "stride", "__weakref__")


class _Saves:
    """What one block of the context has packed so far, while a node holds it.  Autograd keeps ONE tensor for all the nodes that
    save it (an activation is its own node's output and the next one's input); here those nodes share one checkpoint, or two of
    them would take more than a 16-bit tensor itself.  A tensor is the same as long as its storage lives (the entry's weak
    reference keeps the storage's handle, not its memory, from being used again) and its version counter stands still; what is
    packed on one stream, or outside of a capture, is not there for another stream or inside of one."""
    __slots__ = ("entries", "captured")

    def __init__(self):
        self.entries, self.captured = {}, self.capturing()

    @staticmethod
    def capturing():
        return torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing()

    def pack(self, t, build):
        if t.is_cuda and self.capturing() != self.captured:
            return build(t)
        storage = t.untyped_storage()
        key = (storage._cdata, t.storage_offset(), t.dtype, t.is_neg(), t.size(), t.stride(), t._version, hip_lib.get().stream(t))
        entry = self.entries.get(key)
        kept = entry[0]() if entry is not None else None
        if kept is None:
            kept = build(t)
            if isinstance(kept, _Kept):
                self.entries[key] = (weakref.ref(kept, lambda ref: self._drop(key, ref)), StorageWeakRef(storage))
        return kept

    def _drop(self, key, ref):
        entry = self.entries.get(key)
        if entry is not None and entry[0] is ref:
            del self.entries[key]


def _pack(t, least, saves):
    if t.layout != torch.strided or t.dtype not in hip_lib.element_types() or t.numel() < least or _lives_anyway(t):
        return t
    if not t.is_cuda and hip_lib.get().device_only:
        return t
    return saves.pack(t, _keep)


def _keep(t):
    order = sorted(range(t.dim()), key=lambda d: (-t.stride(d), d))
    flat = t.detach().permute(order)
    if not flat.is_contiguous():          # expanded, overlapping or with gaps: as it is
        return t
    k = _Kept()
    k.size, k.stride = t.size(), t.stride()
    n = t.numel()
    # rows of whole blocks where the memory divides into them (else one row, whose last block is short)
    k.kept = checkpoint8(flat.reshape(-1, next((w for w in (4096, 512, 64, 32) if n % w == 0), n)))
    return k


def _unpack(k):
    if not isinstance(k, _Kept):
        return k
    return k.kept.dequantize().view(-1).as_strided(k.size, k.stride)


@contextlib.contextmanager
def activation_checkpoints8(least=65536, enabled=True):
    """Every autograd node built inside keeps the activations it saves (float32, bfloat16, float16; at least ``least`` values) as
    8-bit checkpoints and gets them back when its backward runs, wherever that is; nodes that save the same tensor share one.
    Parameters (trainable or frozen), other leaves that require a gradient, views of either, small, sparse and host tensors are kept
    as they are.  A weight that is no Parameter (a replica's, a detached or a computed one) is an activation here.  Forward values do
    not change; gradients are those at the values that the checkpoints stand for.  In the backward pass a weight is known by its
    memory alone: convolutions inside lay it out anew for each launch (``weight_prep``)."""
    if not enabled:
        yield
        return
    saves = _Saves()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: _pack(t, least, saves), _unpack):
        yield
