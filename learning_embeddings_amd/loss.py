"""Host mirror of network/loss.py for the hot path: MultiLevelCELoss (loss.py:5-38), config 4's criterion.
forward = one fused HIP launch (softmax statistics, loss, gradient) instead of 4 CE calls + autograd."""
import torch

from . import ops


class MultiLevelCELoss(torch.nn.Module):
    def __init__(self, labelmap, level_weights=None, weight=None):
        torch.nn.Module.__init__(self)
        self.labelmap = labelmap
        self.level_weights = [1.0] * len(self.labelmap.levels) if level_weights is None else level_weights
        # per-class weights (loss.py:16-25): one vector over all n_classes, sliced per level by the reference; the sample's term of a
        # level is scaled by its target class's weight (CrossEntropyLoss(weight=..., reduction='none')).  Held as a buffer-like
        # attribute and moved to the logits' device on first use.
        self.weight = None if weight is None else torch.as_tensor(weight, dtype=torch.float32).reshape(-1).contiguous()
        if self.weight is not None and self.weight.numel() != sum(self.labelmap.levels):
            raise ValueError('weight must hold one entry per class (%d), got %d' % (sum(self.labelmap.levels), self.weight.numel()))
        print('==Using the following weights config for multi level cross entropy loss: {}'.format(self.level_weights))

    def forward(self, outputs, labels, level_labels):
        """criterion(outputs [B, n_classes], labels (unused, as in the reference), level_labels [B, L]) -> mean loss."""
        if self.weight is not None and self.weight.device != outputs.device:
            self.weight = self.weight.to(outputs.device)
        return ops.MultiLevelCEFn.apply(outputs, level_labels, list(self.labelmap.levels), list(self.level_weights), self.weight)


# ------------------------------------------------------------------------------------------------ learning from feedback
# The classifier above answers an image with a label path: one class a level, each level a softmax of its own.  These train it on what its answers are worth rather
# than on labels: on which of two paths an annotator preferred, or on a reward per sampled path.  No counterpart in the reference.
#
# A path is int64 [L], the class WITHIN its level as in `level_labels`, -1 (any negative) where it is not known: such an entry counts nowhere.
#
# A training step may be captured into a HIP graph.  As for every captured backward pass, no eager loss of the same parameters may be alive then (delete it, or keep its detach()).

def path_log_probs(outputs, paths, levels):
    """Log-probabilities of label paths.  outputs [R, n_classes] (float32 / bfloat16 / float16), paths [R, L] or [R, G, L] (G paths a row), levels: a labelmap or
    a sequence of level sizes -> float32 of paths' shape, 0 where the entry is negative.  Differentiable in `outputs`.  A class outside its level gives NaN."""
    lv = ops.PathLevels.of(levels)
    if outputs.dim() != 2 or paths.dim() not in (2, 3):
        raise ValueError('outputs must be [rows, n_classes] and paths [rows, L] or [rows, G, L], got %s and %s' % (tuple(outputs.shape), tuple(paths.shape)))
    G = paths.shape[1] if paths.dim() == 3 else 1
    _check_group(G)
    p = ops._paths_arg(paths, (outputs.shape[0],) + ((G,) if paths.dim() == 3 else ()) + (lv.L,), outputs)
    return ops.PathLogProbFn.apply(outputs, p.view(outputs.shape[0], G, lv.L), lv).view(paths.shape)


def _check_group(G):
    if G > ops.MAX_PATHS_PER_ROW:
        raise ValueError('at most %d paths a row, got %d' % (ops.MAX_PATHS_PER_ROW, G))


class PreferenceLoss(torch.nn.Module):
    """Preference of one label path over another, against a reference model:
        reward(path) = beta * sum over its known levels of (log p(class) - reference's log p(class)),   d = reward(chosen) - reward(rejected)
        loss = mean over pairs of (1 - label_smoothing) softplus(-d) + label_smoothing softplus(d)
    forward(outputs, paths, ref_log_probs) -> (loss, rewards [P, 2] -- chosen, rejected -- without gradient):
        one image a pair:   outputs [P, n_classes],  paths and ref_log_probs [P, 2, L]  (chosen first)
        an image each:      outputs [2P, n_classes], paths and ref_log_probs [2P, L]    (the P chosen, then the P rejected)
    ref_log_probs are constants (path_log_probs of the frozen reference); entries of unknown levels are not used."""

    def __init__(self, labelmap, beta=0.1, label_smoothing=0.0):
        super().__init__()
        self.levels = ops.PathLevels.of(labelmap)
        if not 0.0 <= label_smoothing <= 1.0:
            raise ValueError('label_smoothing must be in [0, 1], got %r' % (label_smoothing,))
        self.beta, self.label_smoothing = float(beta), float(label_smoothing)

    def forward(self, outputs, paths, ref_log_probs):
        R, L = outputs.shape[0], self.levels.L
        shared = paths.dim() == 3
        if R == 0 or (not shared and R % 2):
            raise ValueError('a preference loss needs at least one pair (two rows a pair when paths are [2P, L]), got %d rows' % R)
        shape = (R, 2, L) if shared else (R, L)
        p = ops._paths_arg(paths, shape, outputs)
        ref = ops._entries_arg(ref_log_probs, 'ref_log_probs', shape, outputs)
        return ops.PreferenceLossFn.apply(outputs, p, ref, (self.levels, self.beta, self.label_smoothing, shared))


class ClippedPolicyLoss(torch.nn.Module):
    """Policy gradient on a reward per sampled path, ratio clipped, with a KL term against a reference model.  Entry (row, path, level), A the path's advantage:
        rho = exp(log p - old log p),  q = reference's log p - log p
        t = -min(rho A, clip(rho, 1 - clip_low, 1 + clip_high) A) + kl_coef (exp(q) - q - 1)
    reduction 'level': mean of t over all known entries (0 when there are none); 'path': mean over all paths of each path's mean over its known entries.
    forward(outputs [R, n_classes], paths [R, G, L] or [R, L], advantages [R, G] or [R], old_log_probs=None, ref_log_probs=None)
        -> (loss, stats [2] = mean of exp(q) - q - 1, clipped share -- in the same mean, without gradient).
    old_log_probs None: the paths were drawn from this very model (rho = 1).  ref_log_probs None: no KL term (kl_coef must be 0).  Both, and the advantages, are
    constants: no gradient is taken."""

    def __init__(self, labelmap, clip_low=0.2, clip_high=0.2, kl_coef=0.0, reduction='level'):
        super().__init__()
        self.levels = ops.PathLevels.of(labelmap)
        if reduction not in ('level', 'path'):
            raise ValueError("reduction must be 'level' or 'path', got %r" % (reduction,))
        if clip_low < 0 or clip_high < 0:
            raise ValueError('clip bounds must not be negative, got %r, %r' % (clip_low, clip_high))
        self.clip_low, self.clip_high, self.kl_coef, self.reduction = float(clip_low), float(clip_high), float(kl_coef), reduction

    def forward(self, outputs, paths, advantages, old_log_probs=None, ref_log_probs=None):
        R, L = outputs.shape[0], self.levels.L
        if paths.dim() not in (2, 3):
            raise ValueError('paths must be [rows, L] or [rows, G, L], got %s' % (tuple(paths.shape),))
        lead = (R, paths.shape[1]) if paths.dim() == 3 else (R,)
        G = lead[1] if len(lead) == 2 else 1
        _check_group(G)
        if self.kl_coef != 0.0 and ref_log_probs is None:
            raise ValueError('kl_coef %g needs ref_log_probs' % self.kl_coef)
        if R == 0 or G == 0:
            raise ValueError('a policy loss needs at least one path, got %d rows of %d' % (R, G))
        p = ops._paths_arg(paths, lead + (L,), outputs).view(R, G, L)
        adv = ops._entries_arg(advantages, 'advantages', lead, outputs)
        old = None if old_log_probs is None else ops._entries_arg(old_log_probs, 'old_log_probs', lead + (L,), outputs)
        ref = None if ref_log_probs is None else ops._entries_arg(ref_log_probs, 'ref_log_probs', lead + (L,), outputs)
        return ops.PolicyLossFn.apply(outputs, p, adv, old, ref, (self.levels, self.clip_low, self.clip_high, self.kl_coef, self.reduction == 'path'))
