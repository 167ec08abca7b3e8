"""Class / box predictor (mirrors ROIHead/predictor.py:19-49): stock PyTorch-ROCm, or with int8=True one product of 8-bit
integers that trains with straight-through gradients (ops.LinearI8); Int8FasterRCNNPredictor serves what either has
learnt."""
import torch
from torch.nn import Linear, Module

from .. import ops


class FasterRCNNPredictor(Module):
    int8 = False  # for modules pickled whole before there was a choice

    def __init__(self, in_channels, num_classes, int8=False):
        super().__init__()
        self.cls_score = Linear(in_channels, num_classes)
        self.bbox_pred = Linear(in_channels, num_classes * 4)
        self.int8 = int8

    def forward(self, x):
        x = x.flatten(start_dim=1)
        if self.int8:  # one product: x is quantised once
            y = ops.LinearI8.apply(x, torch.cat([self.cls_score.weight, self.bbox_pred.weight]),
                                   torch.cat([self.cls_score.bias, self.bbox_pred.bias]), False)
            return y[:, :self.cls_score.out_features], y[:, self.cls_score.out_features:]
        return self.cls_score(x), self.bbox_pred(x)
