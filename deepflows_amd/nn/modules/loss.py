"""Loss modules — mirror of DeepFlows/nn/modules/loss.py."""
from .. import functional as F
from .module import Module

__all__ = ['NLLLoss', 'MSELoss', 'CrossEntropyLoss', 'LinearCrossEntropyLoss']


class _Loss(Module):
    def __init__(self, reduction: str = 'mean') -> None:
        super().__init__()
        assert reduction in {'mean', 'sum'}
        self.reduction = reduction


class NLLLoss(_Loss):
    def forward(self, input, target):
        return F.nll_loss(input, target, reduction=self.reduction)


class MSELoss(_Loss):
    def forward(self, input, target):
        return F.mse_loss(input, target, reduction=self.reduction)


class CrossEntropyLoss(_Loss):
    def forward(self, input, target):
        return F.cross_entropy(input, target, reduction=self.reduction)


class LinearCrossEntropyLoss(_Loss):
    """CrossEntropyLoss of a Linear layer's output for class indices, without that output (extension: F.linear_cross_entropy).
    criterion = LinearCrossEntropyLoss(model.fc); loss = criterion(features, class_indices).  The layer is a submodule here too:
    list its parameters with the model's or with the criterion's, not with both."""

    def __init__(self, linear, reduction: str = 'mean', ignore_index: int = -100, label_smoothing: float = 0.0) -> None:
        super().__init__(reduction)
        self.linear = linear
        self.ignore_index, self.label_smoothing = ignore_index, label_smoothing

    def forward(self, input, target):
        return F.linear_cross_entropy(input, self.linear.weight, self.linear.bias, target, self.reduction, self.ignore_index,
                                      self.label_smoothing)
