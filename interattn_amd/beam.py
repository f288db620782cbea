"""The end of a beam search's step: the best continuations of every request.  The pages that
follow them are ``pages.reorder_sequences``."""

import torch

from . import _native as N
from .ops import workspace_tensor
from .prompt import device_of, launch

_LOGITS = {torch.float32: N.IA_F32, torch.bfloat16: N.IA_BF16}
MAX_BEAMS = MAX_BEST = 64


def beam_select(logits, scores, n=None, *, done=None, pad_token=0, workspace=None):
    """Of each request's beams x vocabulary continuations the ``n`` best (the number of beams by
    default, 64 at most), best first: ``scores[b, j] + log_softmax(logits[b * beams + j])[v]``,
    equal ones by ``j * vocab + v``.

    ``logits [batch * beams, vocab]`` bf16 or float32 with contiguous rows (any stride between
    them), ``scores [batch, beams]`` float32 (-inf: a beam that offers nothing, as all but the
    first do in the first step), ``done [batch, beams]`` bool: beams that have ended offer
    ``pad_token`` at their score and nothing else, their logits unread.  NaN counts as -inf; a
    row that holds +inf offers nothing.  Where fewer than ``n`` are offered the rest score -inf.

    Returns ``(scores [batch, n] float32, tokens [batch, n] int32, parents [batch, n] int32)``,
    new tensors; parents are rows ``b * beams + j``, as ``reorder_sequences`` takes them.  Keys
    are compared in 64 bits, their logs of sums (of float32 exponentials) off by at most
    2^-24 (14 + 2.3 d), d how far a row's tokens lie under its largest logit on average, by their
    probability (less than log vocab); the same call gives the same bits (how rows are cut, and
    with it a sum's last bits, follows from the sizes).  Launches on the current stream, never
    synchronises, can be captured."""
    device_of(logits, scores, done)
    if scores.dim() != 2 or scores.dtype != torch.float32 or not scores.is_contiguous():
        raise ValueError("scores must be contiguous float32 [batch, beams]")
    batch, beams = scores.shape
    if logits.dim() != 2 or logits.shape[0] != batch * beams or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("logits must be [batch * beams, vocab] with contiguous rows")
    if logits.dtype not in _LOGITS:
        raise ValueError("logits must be bfloat16 or float32")
    vocab = logits.shape[1]
    n = beams if n is None else int(n)
    if not 1 <= beams <= MAX_BEAMS or not 1 <= n <= min(MAX_BEST, beams * vocab):
        raise ValueError(f"beam_select takes 1 to {MAX_BEAMS} beams and the best 1 to {MAX_BEST} of beams * vocab")
    if not 0 <= pad_token < vocab:
        raise ValueError("pad_token must be in the vocabulary")
    if done is not None and (done.shape != scores.shape or done.dtype not in (torch.bool, torch.uint8)
                             or not done.is_contiguous()):
        raise ValueError("done must be contiguous bool [batch, beams]")
    dev, code = logits.device, _LOGITS[logits.dtype]
    best = scores.new_empty((batch, n))
    tokens = scores.new_empty((batch, n), dtype=torch.int32)
    parents = torch.empty_like(tokens)
    if batch == 0:
        return best, tokens, parents
    lib = N.lib()
    key = ("beam_scratch", batch, beams, vocab, n, code)
    ws = None if workspace is None else workspace.get(key)
    if ws is None or ws.device != dev:
        need = lib.ia_beam_select_workspace_size(batch, beams, vocab, n, code)
        if not need:
            raise ValueError("beam_select: batch or vocabulary too large")
        ws = workspace_tensor(workspace, key, (need,), device=dev, dtype=torch.uint8, zero=True)
    launch(lib.ia_beam_select, logits, logits.data_ptr(), code, logits.stride(0) if batch * beams > 1 else vocab,
           scores.data_ptr(), None if done is None else done.data_ptr(), int(pad_token), batch, beams, vocab, n,
           best.data_ptr(), tokens.data_ptr(), parents.data_ptr(), ws.data_ptr(), ws.numel())
    return best, tokens, parents
