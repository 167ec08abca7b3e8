"""Class / box predictor (mirrors ROIHead/predictor.py:19-49): stock PyTorch-ROCm, or with int8=True one product of 8-bit
integers that trains with straight-through gradients (ops.LinearI8); Int8FasterRCNNPredictor serves what either has
learnt."""
import torch
from torch.nn import Linear, Module

from .. import ops
from .int8 import Int8TrainingLinear, as_float, dense, fuses


class FasterRCNNPredictor(Module):
    int8 = False  # for modules pickled whole before there was a choice

    def __init__(self, in_channels, num_classes, int8=False):
        super().__init__()
        layer = Int8TrainingLinear if int8 else Linear
        self.cls_score = layer(in_channels, num_classes)
        self.bbox_pred = layer(in_channels, num_classes * 4)
        self.int8 = int8

    def forward(self, x):
        x = x.flatten(start_dim=1)
        if not self.int8:
            return as_float(self.cls_score)(x), as_float(self.bbox_pred)(x)
        if fuses(self.cls_score) and fuses(self.bbox_pred) and self.cls_score.bias is not None \
                and self.bbox_pred.bias is not None:  # one product: x is quantised once
            y = ops.LinearI8.apply(x, torch.cat([self.cls_score.weight, self.bbox_pred.weight]),
                                   torch.cat([self.cls_score.bias, self.bbox_pred.bias]), False)
            return y[:, :self.cls_score.out_features], y[:, self.cls_score.out_features:]
        return dense(self.cls_score, x), dense(self.bbox_pred, x)
