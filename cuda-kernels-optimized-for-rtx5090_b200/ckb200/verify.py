"""Verification of drafted tokens on B200: run({"target_probs", "draft_tokens", "uniforms"[, "draft_probs",
"num_drafts"]}) -> {"tokens", "accepted"}.

The step after the target model's softmax in speculative decoding: each drafted token is accepted with probability
min(1, p / q), and the token after the accepted ones is drawn from what the target's probabilities exceed the draft's by
(or from the target's own after a full draft), so the tokens are distributed as the target's. The random numbers are
inputs. One kernel, no workspace (ckb_verify_launch); no counterpart in the reference.
"""

import torch

from . import _native

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}


def _problem(target, tokens, uniforms, draft, counts):
    """Why these inputs are not a verification these kernels serve, or None."""
    shape, dtype = target.shape, target.dtype
    if dtype not in _DTYPES or len(shape) != 3 or shape[1] < 1 or shape[2] < 1:
        return f"target_probs {dtype} {tuple(shape)}, fp32 or bf16 [B, K + 1, V] is served"
    batch, rows, vocab = shape
    if vocab > 1 << 30 or rows > 1 << 20:
        return f"target_probs {tuple(shape)}"
    if tokens.dtype != torch.int64 or tokens.shape != (batch, rows - 1):
        return f"draft_tokens {tokens.dtype} {tuple(tokens.shape)} for target_probs {tuple(shape)}"
    if uniforms.dtype != torch.float32 or uniforms.shape != (batch, rows):
        return f"uniforms {uniforms.dtype} {tuple(uniforms.shape)}, float32 {(batch, rows)} is needed"
    if draft is not None and (draft.dtype != dtype or draft.shape != (batch, rows - 1, vocab)):
        return f"draft_probs {draft.dtype} {tuple(draft.shape)} for target_probs {dtype} {tuple(shape)}"
    if counts is not None and (counts.dtype != torch.int64 or counts.shape != (batch,)):
        return f"num_drafts {counts.dtype} {tuple(counts.shape)}, int64 {(batch,)} is needed"
    return None


def _strided(t):
    """t (copied where its last dim is not contiguous) and its first two strides, 0 for a dim of size 1."""
    if t.stride(2) != 1 and t.shape[2] != 1:
        t = t.contiguous()
    batch, row, _ = t.stride()
    return t, 0 if t.shape[0] == 1 else batch, 0 if t.shape[1] == 1 else row


def verify_drafts(target_probs, draft_tokens, uniforms, draft_probs=None, num_drafts=None, out=None):
    """Checks drafted tokens: (tokens [B, K + 1], accepted [B]), int64. Row b of tokens holds the accepted drafted tokens,
    then the newly drawn one, then -1; accepted[b] counts the first.

    target_probs [B, K + 1, V] (fp32 or bf16, as softmax() gives them) are the target's at each drafted place and the one
    after; draft_tokens [B, K] int64; uniforms [B, K + 1] fp32 in [0, 1), the last of a row for the drawing. Token i is
    accepted when uniforms[b, i] * draft_probs[b, i, token] < target_probs[b, i, token]; draft_probs [B, K, V] None
    stands for drafts without probabilities (all mass on the drafted token). num_drafts [B] int64: the drafted tokens
    of each sequence where they differ (clamped to [0, K]). A token outside [0, V) is refused. A NaN or negative
    probability counts as 0; a drawn token is -1 where its row has no mass. Sums are taken in 64 bits. The probabilities
    may be views with any strides whose last dim is contiguous. out = (tokens, accepted) gives the output tensors."""
    problem = _problem(target_probs, draft_tokens, uniforms, draft_probs, num_drafts)
    if problem:
        raise ValueError(f"verify: {problem}")
    given = [t for t in (draft_probs, num_drafts) if t is not None]
    _native.require_cuda("verify", target_probs, draft_tokens, uniforms, *given)
    batch, rows, vocab = target_probs.shape
    if out is None:
        tokens, accepted = draft_tokens.new_empty((batch, rows)), draft_tokens.new_empty((batch,))
    else:
        tokens, accepted = out
        for t, shape in ((tokens, (batch, rows)), (accepted, (batch,))):
            if tuple(t.shape) != shape or t.dtype != torch.int64 or not t.is_contiguous() or \
                    t.device != target_probs.device:
                raise ValueError("verify: out must be contiguous int64 tensors [B, K + 1] and [B] on target_probs' device")
    target, target_batch, target_row = _strided(target_probs)
    draft, draft_batch, draft_row = (None, 0, 0) if draft_probs is None else _strided(draft_probs)
    draft_tokens, uniforms = draft_tokens.contiguous(), uniforms.contiguous()
    counts = None if num_drafts is None else num_drafts.contiguous()
    _native.call(_native.load("verify").ckb_verify_launch, target, target.data_ptr(),
                 None if draft is None else draft.data_ptr(), draft_tokens.data_ptr(),
                 None if counts is None else counts.data_ptr(), uniforms.data_ptr(), tokens.data_ptr(),
                 accepted.data_ptr(), target_batch, target_row, draft_batch, draft_row, batch, rows - 1, vocab,
                 _DTYPES[target.dtype])
    return tokens, accepted


def run(inputs):
    tokens, accepted = verify_drafts(inputs["target_probs"], inputs["draft_tokens"], inputs["uniforms"],
                                     inputs.get("draft_probs"), inputs.get("num_drafts"))
    return {"tokens": tokens, "accepted": accepted}
