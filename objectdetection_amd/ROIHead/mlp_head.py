"""Two-FC head (mirrors ROIHead/mlp_head.py:19-49): stock PyTorch-ROCm, or with int8=True products of 8-bit integers that
train with straight-through gradients (ops.LinearI8); Int8TwoMLPHead serves what either has learnt."""
from torch.nn import Linear, Module, functional

from .int8 import Int8TrainingLinear, as_float, dense_relu


class TwoMLPHead(Module):
    int8 = False  # for modules pickled whole before there was a choice

    def __init__(self, in_channels, representation_size, int8=False):
        super().__init__()
        layer = Int8TrainingLinear if int8 else Linear
        self.fc1 = layer(in_channels, representation_size)
        self.fc2 = layer(representation_size, representation_size)
        self.int8 = int8

    def forward(self, x):
        x = x.flatten(start_dim=1)
        if self.int8:
            return dense_relu(self.fc2, dense_relu(self.fc1, x))
        x = functional.relu(as_float(self.fc1)(x))
        x = functional.relu(as_float(self.fc2)(x))
        return x
