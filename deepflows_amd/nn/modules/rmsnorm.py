"""RMSNorm — root-mean-square normalisation over the last axis, with the residual's addition in front of it on request (the
reference has BatchNorm2d only)."""
from ... import backend_api, tensor
from ...tensor import Tensor
from .. import functional as F
from ..parameter import Parameter
from .module import Module


class RMSNorm(Module):
    def __init__(self, num_features, eps=1e-6, affine=True, device='hip', dtype=None) -> None:
        super().__init__()
        if num_features < 1:
            raise ValueError(f"RMSNorm: num_features must be at least 1, got {num_features}")
        self.num_features, self.eps, self.affine = num_features, eps, affine
        self.weight = Parameter(tensor.ones((num_features,), device=backend_api.Device(device), dtype=dtype)) if affine else None

    def forward(self, x: Tensor, residual: Tensor = None):
        """The normalised x; with `residual` the pair (normalised sum, sum) of x + residual."""
        if int(x.shape[-1]) != self.num_features:
            raise ValueError(f"RMSNorm: a last axis of {self.num_features} is expected, got {tuple(x.shape)}")
        return F.rms_norm(x, self.weight, self.eps, residual)

    def extra_repr(self):
        return f"num_features={self.num_features}, eps={self.eps}, affine={self.affine}"
