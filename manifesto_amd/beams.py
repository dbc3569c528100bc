"""Beam search's selection over beams and vocabulary (include/mfh_beams.h).

Device buffers are integer pointers and streams ``hipStream_t`` integers, as in
``abi``; the descriptor below holds what a program keeps from call to call.
"""
from __future__ import annotations

import ctypes

from .abi import BeamShape, check, lib


class Beams(BeamShape):
    """Shape of a selection: rows of logits are dense unless logits_stride (in elements) is given."""

    def __init__(self, dtype: int, beams: int, picks: int, vocab: int, end_token: int = -1, logits_stride: int = 0,
                 history_stride: int = 0):
        super().__init__()
        self.dtype, self.beams, self.picks, self.vocab, self.end_token = dtype, beams, picks, vocab, end_token
        self.logits_stride, self.history_stride = logits_stride, history_stride


def beam_select_workspace(shape: Beams, groups: int) -> int:
    """Bytes of workspace that beam_select needs."""
    need = ctypes.c_size_t()
    check(lib().mfh_beam_select_workspace(shape, groups, ctypes.byref(need)))
    return need.value


def beam_select(shape: Beams, groups: int, logits: int, scores: int, ended: int, scores_out: int, tokens: int,
                parents: int, ended_out: int, history: int, known: int, history_out: int, workspace: int,
                workspace_bytes: int, stream: int = 0) -> None:
    """The best continuations of each group's beams, best first, and their histories."""
    check(lib().mfh_beam_select(shape, groups, logits, scores, ended, scores_out, tokens, parents, ended_out, history,
                                known, history_out, workspace, workspace_bytes, stream))
