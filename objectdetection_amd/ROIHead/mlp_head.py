"""Two-FC head (mirrors ROIHead/mlp_head.py:19-49): stock PyTorch-ROCm, or with int8=True products of 8-bit integers that
train with straight-through gradients (ops.LinearI8); Int8TwoMLPHead serves what either has learnt."""
from torch.nn import Linear, Module, functional

from .. import ops


class TwoMLPHead(Module):
    int8 = False  # for modules pickled whole before there was a choice

    def __init__(self, in_channels, representation_size, int8=False):
        super().__init__()
        self.fc1 = Linear(in_channels, representation_size)
        self.fc2 = Linear(representation_size, representation_size)
        self.int8 = int8

    def forward(self, x):
        x = x.flatten(start_dim=1)
        if self.int8:
            x = ops.LinearI8.apply(x, self.fc1.weight, self.fc1.bias, True)
            return ops.LinearI8.apply(x, self.fc2.weight, self.fc2.bias, True)
        x = functional.relu(self.fc1(x))
        x = functional.relu(self.fc2(x))
        return x
