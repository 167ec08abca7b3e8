"""The box head's dense layers served in 8-bit integers (ops.linear_i8): the weights of a trained TwoMLPHead /
FasterRCNNPredictor (ROIHead/mlp_head.py:19-49, ROIHead/predictor.py:19-49) quantised once, per output channel; the RoI
features quantised per RoI on every call.  The reference runs these layers in fp32; no counterpart there.

Drop-in for `mlp_head` / `predictor` of ROIHead, and for the padded path (`ROIPooling.forward_padded`): `n_rows`, the
device-side row count, keeps the rows behind it out without a host read.  To train through the same rounding, construct
the float modules with int8=True.
"""
import torch
from torch.nn import Linear, Module, functional
from torch.nn.modules import module as _module

from .. import ops


class Int8TrainingLinear(Linear):
    """torch's Linear with its product on 8-bit integers, differentiable (ops.LinearI8): what TwoMLPHead and
    FasterRCNNPredictor are made of with int8=True.  Same parameters and state_dict.  Takes (M,K)."""

    def forward(self, x):
        return ops.LinearI8.apply(x, self.weight, self.bias, False)


def fuses(layer):
    """Whether a head may compute this layer together with what follows: not where someone watches or changes what goes in
    and out (hooks; weight normalisation as a pre-hook is one), nor another kind of layer put in its place."""
    return (isinstance(layer, Int8TrainingLinear) or type(layer) is Linear) and not (
        layer._forward_hooks or layer._forward_pre_hooks or layer._backward_hooks or layer._backward_pre_hooks
        or _module._global_forward_hooks or _module._global_forward_pre_hooks or _module._global_backward_hooks
        or _module._global_backward_pre_hooks)


def dense(layer, x):
    """layer(x) in 8-bit integers.  A plain Linear (of a head built, or pickled, before it was set to int8) takes the class
    that computes so, which holds the same."""
    if type(layer) is Linear:
        layer.__class__ = Int8TrainingLinear
    return layer(x)


def dense_relu(layer, x):
    """relu(layer(x)) in 8-bit integers, in one call where nothing needs the layer's own output."""
    if fuses(layer):
        return ops.LinearI8.apply(x, layer.weight, layer.bias, True)
    return functional.relu(dense(layer, x))


def as_float(layer):
    """The layer of a head that is not, or no longer, set to int8."""
    if type(layer) is Int8TrainingLinear:
        layer.__class__ = Linear
    return layer


class Int8Linear(Module):
    """y = [relu](x W^T + b) with W as codes (N,K) int8 and scales (N) fp32.  Nothing here is trained: weights change only
    by from_float or load_state_dict.  In eval mode an x that wants a gradient gets it (straight-through), in training mode
    it is refused, lest a head that cannot learn goes unnoticed."""

    def __init__(self, in_features, out_features, bias=True, relu=False):
        super().__init__()
        self.in_features, self.out_features, self.relu = in_features, out_features, relu
        # rows on a stride of 16 bytes, which the kernels read in place
        self.register_buffer("codes", torch.zeros((out_features, (in_features + 15) // 16 * 16), dtype=torch.int8))
        self.register_buffer("scale", torch.zeros((out_features,)))
        self.register_buffer("bias", torch.zeros((out_features,)) if bias else None)

    @classmethod
    def from_float(cls, weight, bias=None, relu=False):
        """weight (N,K) and bias (N) or None, on a HIP device."""
        layer = cls(weight.shape[1], weight.shape[0], bias is not None, relu).to(weight.device)
        codes, scale = ops.quantize_rows_i8(weight.detach())
        layer.codes[:, :weight.shape[1]] = codes
        layer.scale.copy_(scale)
        if bias is not None:
            layer.bias.copy_(bias.detach())
        return layer

    def _apply(self, fn, *args, **kwargs):
        """half(), to(torch.bfloat16) and the like move the buffers but leave the scales and the bias in fp32: a weight's
        scale in fp16 would be a subnormal number."""
        kept = {"scale": self.scale, "bias": self.bias}
        super()._apply(fn, *args, **kwargs)
        for name, t in kept.items():
            now = getattr(self, name)
            if now is not None and now.dtype != t.dtype:
                setattr(self, name, t.to(now.device))
        return self

    def forward(self, x, n_rows=None, out_dtype=None):
        if torch.is_grad_enabled() and x.requires_grad:
            if self.training:
                raise RuntimeError("Int8Linear's weights have no gradient: call eval(), or train TwoMLPHead / "
                                   "FasterRCNNPredictor with int8=True")
            return ops.FrozenLinearI8.apply(x, self.codes[:, :self.in_features], self.scale, self.bias, self.relu, out_dtype,
                                            n_rows)
        return ops.linear_i8(x, self.codes[:, :self.in_features], self.scale, self.bias, self.relu, out_dtype, n_rows)


class Int8TwoMLPHead(Module):
    """TwoMLPHead served in 8-bit integers: flatten -> fc1 -> ReLU -> fc2 -> ReLU, the ReLUs inside the products."""

    def __init__(self, in_channels, representation_size):
        super().__init__()
        self.fc1 = Int8Linear(in_channels, representation_size, relu=True)
        self.fc2 = Int8Linear(representation_size, representation_size, relu=True)

    @classmethod
    def from_float(cls, head):
        layer = cls.__new__(cls)
        Module.__init__(layer)
        layer.fc1 = Int8Linear.from_float(head.fc1.weight, head.fc1.bias, relu=True)
        layer.fc2 = Int8Linear.from_float(head.fc2.weight, head.fc2.bias, relu=True)
        return layer.train(head.training)

    def forward(self, x, n_rows=None):
        return self.fc2(self.fc1(x.flatten(start_dim=1), n_rows), n_rows)


class Int8FasterRCNNPredictor(Module):
    """FasterRCNNPredictor served in 8-bit integers: both of its layers in one product."""

    def __init__(self, in_channels, num_classes):
        super().__init__()
        self.num_classes = num_classes
        self.both = Int8Linear(in_channels, num_classes * 5)

    @classmethod
    def from_float(cls, predictor):
        layer = cls.__new__(cls)
        Module.__init__(layer)
        layer.num_classes = predictor.cls_score.out_features
        layer.both = Int8Linear.from_float(torch.cat([predictor.cls_score.weight, predictor.bbox_pred.weight]),
                                           torch.cat([predictor.cls_score.bias, predictor.bbox_pred.bias]))
        return layer.train(predictor.training)

    def forward(self, x, n_rows=None):
        y = self.both(x.flatten(start_dim=1), n_rows)
        return y[:, :self.num_classes], y[:, self.num_classes:]
