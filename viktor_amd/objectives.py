"""Differentiable objectives on the decoder's logits [B, T, V] at any vocabulary, beside gspo.sequence_ratio_loss
(scripts/gspo.py:474-477) and train.frame_loss (viktor/model.py:153-177):

  token_policy_loss   clipped policy loss per token with a KL term to a reference policy
  preference_loss     loss of paired log ratios: a preferred call against a lesser one
  distill_loss        divergence from a teacher's list of top logits (hip_ops.top_logits)

Each is one autograd node whose forward computes the gradient beside the loss, in the logits' type: a row of logits is read
once and its gradient written once. The first backward hands that gradient out; where the loss's own gradient is not 1 (a
scaled or summed loss) the kernel runs again with that factor in its place, so that the result is rounded once. It looks at
the factor on the device: nothing waits. A second backward through a kept graph computes the gradient anew, and so does one
that is captured without its forward. (One captured in a graph of its own, apart from its forward's, is replayed once for each
replay of that.)
"""

import torch
from torch.autograd.function import once_differentiable

from . import hip_ops as ops


_capturing = torch.cuda.is_current_stream_capturing


class _Objective(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, op, outputs, args, grad):
        res, launch = op(logits.detach(), *args, grad)
        if grad:
            ctx.save_for_backward(logits, *launch.keep(logits))
            ctx.launch, ctx.dlogits, ctx.captured = launch, res["dlogits"], _capturing()
        others = [res[name] for name in outputs]
        ctx.mark_non_differentiable(*(t for t in others if t is not None))
        ctx.set_materialize_grads(False)
        return (res["loss"], *others)

    @staticmethod
    @once_differentiable
    def backward(ctx, g_loss, *unused):
        if g_loss is None:
            return None, None, None, None, None
        logits, *tensors = ctx.saved_tensors  # (raises if an input has been written to since)
        dl, ctx.dlogits = ctx.dlogits, None   # (handed out once: a caller may keep it as its gradient)
        # (a backward captured without its forward writes the gradient at every replay: nothing else would)
        there = dl is not None and ctx.captured == _capturing()
        if dl is None:
            dl = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        ctx.launch.again(logits, tensors, dl, g_loss, there)
        return dl, None, None, None, None


def _objective(logits, op, outputs, args):
    return _Objective.apply(logits, op, outputs, args, logits.requires_grad and torch.is_grad_enabled())


def token_policy_loss(logits, targets, mask, old_lp, adv, ref_lp=None, eps_lo=0.2, eps_hi=0.2, kl_coef=0.0, per="sequence",
                      inv_n=None):
    """hip_ops.policy_score, differentiable in logits: (loss, pg, kl, lp); kl is None without ref_lp. The per-token
    counterpart of gspo.sequence_ratio_loss. pg, kl and lp are values to read."""
    return _objective(logits, ops._policy, ("pg", "kl", "lp"),
                            (targets, mask, old_lp, adv, ref_lp, eps_lo, eps_hi, kl_coef, per, inv_n))


def preference_loss(logits, targets, mask, ref_lp=None, pairs=None, beta=0.1, target=0.0, smoothing=0.0, lengths=None,
                    inv_n=None):
    """hip_ops.preference_score, differentiable in logits: (loss, margin, lp). margin and lp are values to read."""
    return _objective(logits, ops._preference, ("margin", "lp"),
                            (targets, mask, ref_lp, pairs, beta, target, smoothing, lengths, inv_n))


def distill_loss(logits, values, ids, t_lse=None, weights=None, temperature=1.0, inv_n=None):
    """hip_ops.distill_score, differentiable in logits: (loss, kl). kl is a value to read."""
    return _objective(logits, ops._distill, ("kl",), (values, ids, t_lse, weights, temperature, inv_n))
