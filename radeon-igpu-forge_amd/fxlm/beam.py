"""fxlm.beam: the selection of a beam search's step.

The reference samples one token a pass (its ml/fxlm/sample.py:62-73) and has no beams.  Inference:
what comes out has no gradient.
"""
import torch

from fxgpu.abi import host

from .speculative import _taken


def beam_select(logits, scores, done=None, fill=0, weight=None):
    """The best K continuations of each sequence's K beams by one token.

    logits (B, K, V) fp32 or bf16 cuda: a beam's logits for its next token; scores (B, K) fp32: the
    beams' sums of log-probabilities, -inf for one that does not exist (its logits are not read).  A
    beam's continuation by token v has the score scores[b, k] + log_softmax(logits[b, k])[v].  done
    (B, K) bool: a beam that has ended goes on as it is, by the token `fill`, its score unchanged.
    weight (B, K) fp32, positive and finite: continuations are ranked by weight times score (a length penalty).
    A token whose logit is -inf continues nothing.  K <= 32, V <= 1,048,576.

    Returns, best first, scores (B, K) fp32; parents (B, K) int32, the row b * K + k that each goes on
    from (reorder_pages' parents); tokens (B, K) int64.  Equal ranks go to the lower beam, then to the
    larger logit, then to the lower token.  Log-probabilities come from sums in 32 bits, off by 1e-5 at
    most and by 1e-7 as a rule: unlike beams' continuations that are nearer than that may come in either
    order; beams of equal logits and scores rank alike.  Where there are fewer than K continuations the
    rest have score -inf, parent -1 and token `fill`.  A beam whose score or log-probabilities are not numbers
    (a NaN or +inf among its logits), or whose weight is not positive and finite, has one continuation, of
    score NaN and token `fill`, and NaN ranks first: it is not lost silently.
    """
    r = host.beam_select(logits, scores, done, int(fill), weight)
    if r is None:
        if logits.dim() != 3:
            raise ValueError(f"logits must be (B, K, V), got {tuple(logits.shape)}")
        B, K, V = logits.shape
        if B < 1 or not 1 <= K <= 32 or not 1 <= V <= 1048576:
            raise ValueError(f"logits {tuple(logits.shape)}: 1 to 32 beams, a vocabulary of 1 to 1,048,576")
        if logits.dtype not in (torch.float32, torch.bfloat16):
            raise TypeError(f"logits must be float32 or bfloat16, got {logits.dtype}")
        for nm, t, want in (("logits", logits, logits.dtype), ("scores", scores, torch.float32), ("done", done, torch.bool),
                            ("weight", weight, torch.float32)):
            if t is None:
                continue
            if t.dtype != want:
                raise TypeError(f"{nm} must be {want}, got {t.dtype}")
            if not t.is_cuda:
                raise TypeError(f"{nm} must be a cuda tensor")
            if tuple(t.shape[:2]) != (B, K) or (t is not logits and t.dim() != 2):
                raise ValueError(f"{nm} must be {(B, K)}, got {tuple(t.shape)}")
        x = logits.contiguous()   # a slice of positions, or rows at an odd address
        r = host.beam_select(x if x.data_ptr() % 16 == 0 else x.clone(), scores.contiguous(), None if done is None else done.contiguous(), int(fill),
                             None if weight is None else weight.contiguous())
    return _taken(r, "beam_select")
