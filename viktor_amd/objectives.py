"""Differentiable objectives on the decoder's logits [B, T, V] at any vocabulary, beside gspo.sequence_ratio_loss
(scripts/gspo.py:474-477) and train.frame_loss (viktor/model.py:153-177):

  token_policy_loss   clipped policy loss per token with a KL term to a reference policy
  preference_loss     loss of paired log ratios: a preferred call against a lesser one
  distill_loss        divergence from a teacher's list of top logits (hip_ops.top_logits)

Each is one autograd node whose forward computes the gradient beside the loss, in the logits' type: a row of logits is read
once and its gradient written once. The first backward hands that gradient out; where the loss's own gradient is not 1 (a
scaled or summed loss) the kernel runs again with that factor in its place, so that the result is rounded once. It looks at
the factor on the device: nothing waits. A second backward through a kept graph computes the gradient anew.
"""

import torch
from torch.autograd.function import once_differentiable

from . import hip_ops as ops


class _Objective(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, op, outputs, tensors, options):
        res = op(logits.detach(), **tensors, **options, grad=ctx.needs_input_grad[0])
        ctx.op, ctx.options, ctx.names = op, options, list(tensors)
        ctx.dlogits, ctx.workspace = res.get("dlogits"), res.get("workspace")
        ctx.save_for_backward(logits, *tensors.values())
        others = tuple(res[name] for name in outputs)
        ctx.mark_non_differentiable(*(t for t in others if t is not None))
        ctx.set_materialize_grads(False)
        return (res["loss"], *others)

    @staticmethod
    @once_differentiable
    def backward(ctx, g_loss, *unused):
        logits, *tensors = ctx.saved_tensors
        if g_loss is None:
            return None, None, None, None, None
        more = {} if ctx.workspace is None else {"workspace": ctx.workspace}
        dl, ctx.dlogits = ctx.dlogits, None  # (handed out once: a caller may keep it as its gradient)
        if dl is not None:
            more |= {"out": dl, "unless_one": True}
        res = ctx.op(logits.detach(), **dict(zip(ctx.names, tensors)), **ctx.options, **more, upstream=g_loss.float())
        return res["dlogits"], None, None, None, None


def token_policy_loss(logits, targets, mask, old_lp, adv, ref_lp=None, eps_lo=0.2, eps_hi=0.2, kl_coef=0.0, per="sequence",
                      inv_n=None):
    """hip_ops.policy_score, differentiable in logits: (loss, pg, kl, lp); kl is None without ref_lp. The per-token
    counterpart of gspo.sequence_ratio_loss. pg, kl and lp are values to read."""
    return _Objective.apply(logits, ops.policy_score, ("pg", "kl", "lp"),
                            {"targets": targets, "mask": mask, "old_lp": old_lp, "adv": adv, "ref_lp": ref_lp},
                            {"eps_lo": eps_lo, "eps_hi": eps_hi, "kl_coef": kl_coef, "per": per, "inv_n": inv_n})


def preference_loss(logits, targets, mask, ref_lp=None, pairs=None, beta=0.1, target=0.0, smoothing=0.0, lengths=None,
                    inv_n=None):
    """hip_ops.preference_score, differentiable in logits: (loss, margin, lp). margin and lp are values to read."""
    return _Objective.apply(logits, ops.preference_score, ("margin", "lp"),
                            {"targets": targets, "mask": mask, "ref_lp": ref_lp, "pairs": pairs, "lengths": lengths},
                            {"beta": beta, "target": target, "smoothing": smoothing, "inv_n": inv_n})


def distill_loss(logits, values, ids, t_lse=None, weights=None, temperature=1.0, inv_n=None):
    """hip_ops.distill_score, differentiable in logits: (loss, kl). kl is a value to read."""
    return _Objective.apply(logits, ops.distill_score, ("kl",),
                            {"values": values, "ids": ids, "t_lse": t_lse, "weights": weights},
                            {"temperature": temperature, "inv_n": inv_n})
