"""Tuning a summariser from preferences and rewards: scoring given summaries, the paired preference loss, the clipped policy loss with a KL
term, and the scaled embedding with its reproducible gradient.

Logits are [N, T, V] (f32 or bf16; a view of a padded buffer will do), labels int64 [N, T]; a label outside 0 .. V-1 (-100, say) marks a
position that does not count.  Two forms of each loss: a module whose result goes into a larger autograd graph, and a fused call that turns
logits into loss and gradient at once, as the fused training step does with its label-smoothing loss (`dlogits=logits` writes the gradient
over the logits, which are gone then: a backward pass that saved them raises, as after any change in place).
"""
import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import kernels as kn


def _constant(**tensors):
    for name, t in tensors.items():
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise ValueError("%s gets no gradient: detach it" % name)


def sequence_logprobs(logits, labels, average=False):
    """(sum or mean log-probability of every sequence [N], log-probability of every token [N, T]) under the logits; no autograd."""
    logits = logits.detach()
    logp = kn.token_logprob(logits, labels)
    return kn.sequence_logprob(logp, labels, logits.shape[2], average), logp


def preference_loss_and_grad(logits, labels, ref_logps=None, *, beta=0.1, label_smoothing=0.0, average=False, dlogits=None):
    """Paired preference loss of [chosen; rejected] sequences (the first N / 2 and the last) and its gradient:
    h = beta ((S_c - ref_c) - (S_r - ref_r)), loss = mean (1 - e) softplus(-h) + e softplus(h), S the sum (average: mean) of a sequence's
    counted log-probabilities, ref_logps f32 [N] the frozen model's (None: zeros).  -> (loss, margins h [N / 2], dlogits)."""
    loss, margins, _, dlogits = kn.preference_loss(logits.detach(), labels, ref_logps, beta, label_smoothing, average, dlogits)
    return loss, margins, dlogits


def policy_loss_and_grad(logits, labels, old_logps, advantages, ref_logps=None, *, clip_low=0.2, clip_high=0.2, kl_coef=0.0, reduction="token", dlogits=None):
    """Clipped policy loss of sampled sequences and its gradient, the logits read once:
    token loss = max(-A r, -A clip(r, 1 - clip_low, 1 + clip_high)) + kl_coef (e^d - d - 1), r = exp(logp - old_logps), d = ref_logps - logp;
    the mean over all counted tokens ("token") or over the sequences' means ("sequence"); with kl_coef 0 the KL estimate is only reported.
    old_logps, ref_logps f32 [N, T], advantages f32 [N] or [N, T].  -> (loss, mean KL estimate, share of clipped tokens, logp [N, T], dlogits)."""
    out, logp, dlogits = kn.policy_loss(logits.detach(), labels, old_logps, advantages, ref_logps, clip_low, clip_high, kl_coef, reduction, dlogits)
    loss, kl, clipped = out.unbind(0)
    return loss, kl, clipped, logp, dlogits


class _PreferenceFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, ref, beta, smoothing, average):
        stats = torch.empty(*logits.shape[:2], 2, dtype=torch.float32, device=logits.device)
        logp = kn.token_logprob(logits, labels, stats)
        loss, margins, seq, coef = kn.preference_pairs(logp, labels, ref, logits.shape[2], beta, smoothing, average)
        ctx.save_for_backward(logits, labels, stats, coef)
        ctx.mark_non_differentiable(margins, seq)
        return loss, margins, seq

    @staticmethod
    @once_differentiable
    def backward(ctx, g, _margins, _seq):
        logits, labels, stats, coef = ctx.saved_tensors
        return kn.token_logprob_bwd(logits, labels, stats, coef, alpha=g.contiguous()), None, None, None, None, None


class PreferenceLoss(nn.Module):
    """preference_loss_and_grad as a module: forward -> loss, differentiable with respect to the logits.  `margins` [N / 2] and `logps` [N] of the
    last call are kept for monitoring."""

    def __init__(self, beta=0.1, label_smoothing=0.0, average=False):
        super().__init__()
        self.beta, self.label_smoothing, self.average = float(beta), float(label_smoothing), bool(average)
        self.margins = self.logps = None

    def forward(self, logits, labels, ref_logps=None):
        _constant(ref_logps=ref_logps)
        loss, self.margins, self.logps = _PreferenceFn.apply(logits, labels, ref_logps, self.beta, self.label_smoothing, self.average)
        return loss


class _PolicyFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, old, adv, ref, low, high, kl_coef, reduction):
        stats = torch.empty(*logits.shape[:2], 2, dtype=torch.float32, device=logits.device)
        logp = kn.token_logprob(logits, labels, stats)
        out, coef = kn.policy_terms(logp, labels, old, adv, ref, logits.shape[2], low, high, kl_coef, reduction)
        ctx.save_for_backward(logits, labels, stats, coef)
        loss, kl, clipped = out[0].clone(), out[1].clone(), out[2].clone()
        ctx.mark_non_differentiable(kl, clipped, logp)
        return loss, kl, clipped, logp

    @staticmethod
    @once_differentiable
    def backward(ctx, g, *_):
        logits, labels, stats, coef = ctx.saved_tensors
        return (kn.token_logprob_bwd(logits, labels, stats, coef, alpha=g.contiguous()),) + (None,) * 8


class ClippedPolicyLoss(nn.Module):
    """policy_loss_and_grad as a module: forward -> loss, differentiable with respect to the logits.  `kl`, `clipped` and `logps` [N, T] of the last
    call are kept for monitoring."""

    def __init__(self, clip_low=0.2, clip_high=0.2, kl_coef=0.0, reduction="token"):
        super().__init__()
        self.clip_low, self.clip_high, self.kl_coef, self.reduction = float(clip_low), float(clip_high), float(kl_coef), reduction
        self.kl = self.clipped = self.logps = None

    def forward(self, logits, labels, old_logps, advantages, ref_logps=None):
        _constant(old_logps=old_logps, advantages=advantages, ref_logps=ref_logps)
        loss, self.kl, self.clipped, self.logps = _PolicyFn.apply(logits, labels, old_logps, advantages, ref_logps, self.clip_low, self.clip_high, self.kl_coef,
                                                                  self.reduction)
        return loss


def scaled_embedding_grad(dy, ids, num_embeddings, scale=1.0, padding_idx=None, out=None, accumulate=False):
    """Gradient f32 [num_embeddings, D] of scaled_embedding's table, summed by sorted tokens (the same bits on every run); accumulate: added to `out`,
    whose other rows stay as they were."""
    return kn.embed_bwd(dy.detach(), ids, int(num_embeddings), scale, padding_idx, out, accumulate)


class _EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, scale, padding_idx):
        ctx.save_for_backward(ids)
        ctx.V, ctx.scale, ctx.padding_idx, ctx.dtype = table.shape[0], scale, padding_idx, table.dtype
        return kn.embed_fwd(ids, table, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        (ids,) = ctx.saved_tensors
        return None, kn.embed_bwd(dy, ids, ctx.V, ctx.scale, ctx.padding_idx).to(ctx.dtype), None, None


def scaled_embedding(ids, table, scale=1.0, padding_idx=None):
    """scale * table[ids] (f32 or bf16 table, int64 ids of any shape; ids outside the table give zero rows), differentiable with respect to the table
    (padding_idx: a row without a gradient, negative ones counted from the end)."""
    padding_idx = kn.padding_row(padding_idx, table.shape[0])
    kn.no_tangent(table, "scaled_embedding")
    if table.requires_grad and torch.is_grad_enabled():
        return _EmbeddingFn.apply(ids, table, float(scale), padding_idx)
    return kn.embed_fwd(ids, table, float(scale))


class ScaledEmbedding(nn.Module):
    """An embedding whose rows are multiplied by `scale` on the way out (sqrt(d_model), say)."""

    def __init__(self, num_embeddings, embedding_dim, scale=1.0, padding_idx=None, device="cuda", dtype=torch.float32):
        super().__init__()
        self.scale, self.padding_idx = float(scale), kn.padding_row(padding_idx, num_embeddings)
        self.weight = nn.Parameter(torch.empty(num_embeddings, embedding_dim, device=device, dtype=dtype))
        nn.init.normal_(self.weight, std=0.02)
        if padding_idx is not None:
            with torch.no_grad():
                self.weight[self.padding_idx].zero_()

    def forward(self, ids):
        return scaled_embedding(ids, self.weight, self.scale, self.padding_idx)
