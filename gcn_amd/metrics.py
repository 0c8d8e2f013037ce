"""Masked loss and accuracy of the reference (gcn/metrics.py:85-101) on GPU tensors."""
import torch
from torch.autograd.function import once_differentiable

from . import layers, sparse


def masked_softmax_cross_entropy(preds, labels, mask):
    """Softmax cross-entropy with masking: mean over ALL rows of CE_i * mask_i / mean(mask)
    (gcn/metrics.py:85-92).  ``labels`` may hold all-zero rows (CiteSeer's padded nodes): their
    cross-entropy is 0, as tf.nn.softmax_cross_entropy_with_logits gives."""
    labels = labels.to(torch.float32)
    loss = -(labels * torch.log_softmax(preds, dim=1)).sum(dim=1)
    mask = mask.to(torch.float32)
    mask = mask / mask.mean()
    return (loss * mask).mean()


def masked_accuracy(preds, labels, mask):
    """Accuracy with masking (gcn/metrics.py:94-101); argmax of an all-zero label row is 0."""
    correct = (torch.argmax(preds, 1) == torch.argmax(labels, 1)).to(torch.float32)
    mask = mask.to(torch.float32)
    mask = mask / mask.mean()
    return (correct * mask).mean()


class _DistillationFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, preds, values, indices, mask, mask_mean, temperature):
        stats, _ = sparse.distill_topk(preds, values, indices, mask, mask_mean, temperature=temperature, want_grad=False)
        with sparse._on_device(stats):        # loss_summary enqueues on the current device's stream
            loss, agreement = sparse.loss_summary(stats, None, 0.0).unbind()
        ctx.save_for_backward(preds, values, indices, mask)
        ctx.mask_mean, ctx.temperature = mask_mean, temperature
        ctx.mark_non_differentiable(agreement)
        return loss, agreement

    @staticmethod
    @once_differentiable
    def backward(ctx, grad, _):
        preds, values, indices, mask = ctx.saved_tensors
        _, d = sparse.distill_topk(preds, values, indices, mask, ctx.mask_mean, temperature=ctx.temperature,
                                   want_stats=False, upstream=grad.float().contiguous())
        return d, None, None, None, None, None


def masked_distillation(preds, values, indices, mask=None, temperature=1.0, mask_mean=None):
    """(loss, agreement) of a model that learns from a teacher's top logits under the reference's mask: the mean over ALL
    rows of ``T^2 KL(teacher || student) * mask_i / mean(mask)``, and the same mean of whether the two arg maxima are the
    same class.  ``values`` [n x k] are the teacher's logits of the classes ``indices`` (int32, or int64 as ``torch.topk``
    returns them; outside the classes: no entry), as ``sparse.distill_topk`` takes them.  ``mask`` [n]: bool, as the
    reference's are, or whole numbers that weigh the rows.  Differentiable in ``preds``: the backward pass reads the logits
    again instead of keeping a gradient of their size (2^22 x 47: 662 us for both passes, 382 for ``sparse.distill_topk``,
    which gives loss rows and gradient in one).  ``mask_mean``: mean(mask) as a number,
    if the caller has it -- taking it here waits for the device, which a recorded call cannot."""
    held = layers._accumulators(preds)        # noqa: F841 -- alive until the call below has its graph
    if mask is not None and not (mask.is_floating_point() or mask.is_complex()):
        mask = mask.to(torch.int32)
    if indices.dtype == torch.int64:          # what int32 does not hold is no class either
        indices = indices.clamp(-1, 2 ** 31 - 1).to(torch.int32)
    if mask_mean is None:
        mask_mean = 1.0 if mask is None else float(mask.to(torch.float32).mean().item())
    return _DistillationFn.apply(preds, values, indices, mask, float(mask_mean), float(temperature))
