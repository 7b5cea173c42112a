import torch
import torch.nn as nn

from morphocore_b200.functional import rms_norm


class RMSNorm(nn.Module):
    """Root-mean-square norm over the channels with a learnable factor a channel (ones at first) and an optional residual. See
    `morphocore_b200.functional.rms_norm` for the arguments and for what `forward` returns."""

    def __init__(self, num_channels: int, eps: float = 1e-6, dim: int = -3, output: str = "float", dtype: torch.dtype = torch.float32):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(num_channels, dtype=dtype))
        self.eps = eps
        self.dim = dim
        self.output = output

    def forward(self, x: torch.Tensor, residual: torch.Tensor = None):
        return rms_norm(x, self.weight, residual, self.eps, self.dim, self.output)
