"""Layer normalisation as a module: nn.LayerNorm's constructor, parameters and state_dict, the HIP kernels' forward and backward pass
(csrc/layer_norm.hip).  Unlike BatchNorm its statistics are a row's own: one sample trains like many, and data-parallel shards agree without
an exchange."""
import torch.nn as nn

from . import ops


class LayerNorm(nn.LayerNorm):
    """nn.LayerNorm over the last axes.  float32, float16 and bfloat16 input; parameters in float32 or the input's type.  The output has the input's
    type, under autocast too (nn.LayerNorm returns float32 there): statistics and arithmetic are fp32 whatever the types."""

    def forward(self, x):
        n = len(self.normalized_shape)
        if tuple(x.shape[x.ndim - n:]) != tuple(self.normalized_shape):
            raise ValueError(f"LayerNorm over {tuple(self.normalized_shape)}: input of shape {tuple(x.shape)}")
        w, b = self.weight, self.bias
        if n == 1:
            return ops.layer_norm(x, w, b, self.eps)
        flat = ops.layer_norm(x.flatten(x.ndim - n), None if w is None else w.flatten(), None if b is None else b.flatten(), self.eps)
        return flat.view(x.shape)
