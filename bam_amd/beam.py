"""Beam search's selection: of the continuations of a request's beams by a token, those with the largest sums of log-probabilities.

The sequences that go on behind it are reordered by KVCache.reorder.  The reference has no counterpart; the C-ABI is bam_beam_select of include/bam_amd.h.
"""
import ctypes
import struct

import torch
from torch.autograd import forward_ad

from . import _lib
from .host import BamError, _chk, _current, _raw_stream, _stream, _wants_gradients, c_u64, c_vp

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_SELECT = struct.Struct("@QQQPqPqPPPPQIi")          # bam_beam_select_t
_bytes = {}


def beam_select(logits, scores, width=None):
    """The best continuations of each request's beams: (sums, beams, tokens), [requests, width] each, in float32, int32 and int32, the largest sum first.

    logits: [requests * beams, vocab] in bfloat16, float16 or float32, a request's beams one after the other; scores: [requests, beams] in float32, the sum of log-probabilities of each
    beam so far.  sum = score + logit - log(sum(exp(logits of the beam))); `beams` are rows of logits.  Equal sums: the lower beam first, then the lower token.  Tokens of a beam are
    in the order of sums in 64 bits, those of different beams where their sums differ by more than 2^-18 (exponentials are taken in 32 bits).  width: beams unless given,
    256 at most.  A beam whose score is minus infinity has no finite continuation; one with NaN or infinity among its logits, or nothing above minus infinity, has NaN, which comes last.
    There are no gradients: tensors that require them are refused where gradients are being recorded, and those with a tangent (forward_ad).  Queued on the current stream of the tensors' device."""
    shape, beams = logits.shape, scores.shape
    kind, index = _TYPES.get(logits.dtype), logits.get_device()
    if kind is None or len(shape) != 2 or index < 0:
        raise BamError("beam_select: logits must be [requests * beams, vocab] in bfloat16, float16 or float32 on the device")
    if len(beams) != 2 or scores.dtype is not torch.float32 or scores.get_device() != index or beams[0] * beams[1] != shape[0] or beams[1] < 1:
        raise BamError(f"beam_select: scores must be [requests, beams] in float32 on {logits.device}, with a beam for each row of logits")
    row, one = logits.stride()
    score_row, next_score = scores.stride()
    if (one != 1 and shape[1] > 1) or (next_score != 1 and beams[1] > 1):
        raise BamError("beam_select: the numbers of a row must be next to each other")
    if (logits.requires_grad or scores.requires_grad or forward_ad._current_level >= 0) and (_wants_gradients(logits) or _wants_gradients(scores)):
        raise BamError("beam_select: there are no gradients: detach what requires them or has a tangent, or call under torch.no_grad()")
    if width is None:
        width = beams[1]
    if type(width) is not int or not 1 <= width <= 256:
        raise BamError("beam_select: width must be a number from 1 to 256")
    key = (*beams, shape[1], width, kind)
    need = _bytes.get(key)
    L = _lib.load()
    if need is None:
        b = c_u64(0)
        _chk(L.bam_beam_select_bytes(*key, ctypes.byref(b)), "bam_beam_select_bytes")
        if len(_bytes) > 4096:
            _bytes.clear()
        need = _bytes[key] = b.value
    if _current() != index:
        with torch.cuda.device(index):
            return _select(L, logits, scores, row, score_row, beams, width, kind, need)
    return _select(L, logits, scores, row, score_row, beams, width, kind, need)


def _select(L, logits, scores, row, score_row, beams, width, kind, need):
    device = logits.device
    # (one tensor and its parts take less than three.)  The workspace is from torch's allocator, which keeps it for this stream, or for the graph that is being captured
    out, work = torch.empty((3, beams[0], width), dtype=torch.int32, device=device), torch.empty(need, dtype=torch.uint8, device=device)
    if beams[0]:
        at, each = out.data_ptr(), 4 * beams[0] * width
        what = _SELECT.pack(beams[0], beams[1], logits.shape[1], logits.data_ptr(), row, scores.data_ptr(), score_row, at, at + each, at + 2 * each, work.data_ptr(), need, width, kind)
        # (the device is up, there are tensors on it: _stream asks for that first, 0.2 us)
        _chk(L.bam_beam_select(what, c_vp(_raw_stream(device.index)) if _raw_stream is not None else _stream()), "bam_beam_select")
    sums, chosen, tokens = out.unbind(0)
    return sums.view(torch.float32), chosen, tokens
