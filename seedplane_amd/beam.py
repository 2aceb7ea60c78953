"""Beam search's selection on MI355X: the best continuations of each request's beams, in one pass over the logits.

    step = beam_select(logits, scores, eos=eos)             # logits [requests * beams, vocabulary], scores [requests, beams]
    pool.fork(step.next_rows.view(-1))                      # the beams' pages follow (seedplane_amd.pages)
    scores, tokens = step.next_scores, step.next_tokens

Everything runs on torch's current stream of the logits' device, without waiting for it, and may be captured into a graph.  The reference
samples one continuation (seedplane/qwen_engine.py:138-153); it has no beams.
"""
import ctypes
from typing import NamedTuple

import torch

from . import _lib
from .paged import _FLOATS, _call

MOST = 64                                                   # beams, and continuations asked for


class BeamStep(NamedTuple):
    """The best continuations of each request in order, [requests, n], and those of them that go on, [requests, beams]: fp32 scores,
    int32 beams or rows of the logits, int32 tokens; -infinity and -1 in places without one."""
    scores: torch.Tensor
    beams: torch.Tensor
    tokens: torch.Tensor
    next_scores: torch.Tensor
    next_rows: torch.Tensor
    next_tokens: torch.Tensor

    @classmethod
    def allocate(cls, requests, beams, n, device='cuda'):
        a, b, c = torch.empty((3, requests, n), dtype=torch.int32, device=device).unbind(0)
        d, e, f = torch.empty((3, requests, beams), dtype=torch.int32, device=device).unbind(0)
        return cls(a.view(torch.float32), b, c, d.view(torch.float32), e, f)


def beam_select(logits, scores, n=None, eos=None, out=None):
    """The n best of scores[b, k] + log_softmax(logits[b * beams + k]) over beams and vocabulary of each request b, and the best of
    them that do not end, as many as there are beams.

    logits: [requests * beams, vocabulary], fp32, fp16 or bf16, the values of a row side by side; scores: fp32 [requests, beams],
    -infinity for beams that do not live (all but one in a first step).  eos: a token or a list of up to 8 that end a sequence.
    n: default beams * (1 + number of eos), enough for as many to go on as there are beams; at most 64.  Ties go to the lowest beam, then token; logits
    of -infinity, and beams whose logits hold NaN or +infinity, have no continuation.  out: a BeamStep to fill."""
    dt, shape, stride, dev = _FLOATS.get(logits.dtype), logits.shape, logits.stride(), logits.device
    if dt is None or len(shape) != 2 or dev.type != 'cuda' or (stride[1] != 1 and shape[1] > 1):
        raise ValueError('logits must be an fp32, fp16 or bf16 GPU tensor [requests * beams, vocabulary], the values of a row side by side')
    rows, vocab = shape
    if scores.dtype is not torch.float32 or scores.dim() != 2 or scores.device != dev or not scores.is_contiguous() or scores.numel() != rows:
        raise ValueError(f'scores must be a contiguous fp32 tensor [requests, beams] on {dev}, one for each row of the logits')
    requests, beams = scores.shape
    ends = () if eos is None else (eos,) if isinstance(eos, int) else tuple(eos)
    if n is None:
        n = beams * (1 + len(ends))
    if not 1 <= beams <= n <= MOST:
        raise ValueError(f'beams must be in [1, n] and n at most {MOST}; got {beams} and {n}')
    if any(not 0 <= e < 1 << 31 for e in ends):
        raise ValueError('eos must be tokens')
    if out is None:
        out = BeamStep.allocate(requests, beams, n, dev)
    else:
        for i, x in enumerate(out):
            if x.shape != (requests, n if i < 3 else beams) or x.dtype != (torch.int32 if i % 3 else torch.float32) or x.device != dev \
                    or not x.is_contiguous():
                raise ValueError('out must be a BeamStep of these requests, beams and n (BeamStep.allocate)')
    if not requests:
        return out
    lib = _lib.load()
    workspace = torch.empty(lib.sp_op_beam_select_workspace(requests, beams, vocab, n), dtype=torch.uint8, device=dev)
    a, b, c, d, e, f = out
    _call(lib.sp_op_beam_select, dev, dt, logits.data_ptr(), stride[0] if rows > 1 else vocab, requests, beams, vocab, scores.data_ptr(), n,
          len(ends), (ctypes.c_int32 * len(ends))(*ends) if ends else None, a.data_ptr(), b.data_ptr(), c.data_ptr(), d.data_ptr(),
          e.data_ptr(), f.data_ptr(), workspace.data_ptr())
    return out
