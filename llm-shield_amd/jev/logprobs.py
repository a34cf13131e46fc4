"""Log probabilities of rows of logits over libjev's jev_logprobs_* entry points: of given tokens and of
the most probable ones, with the rows' entropy, in one pass on the device (include/jev.h has the rules)."""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import numpy as np

from . import _lib as L


class TokenLogProbs(NamedTuple):
    """Of each row: its given tokens' log probabilities, its entropy, its most probable tokens and theirs."""
    logp: np.ndarray      # [rows][given]
    entropy: np.ndarray   # [rows]
    top: np.ndarray       # [rows][top]
    top_logp: np.ndarray  # [rows][top]


class LogProbs:
    """For calls of up to `max_rows` rows of `vocab` logits.

    logprobs_device takes device pointers (integers) and only enqueues on the handle's stream."""

    def __init__(self, vocab: int, max_rows: int, device: int = 0):
        self._h = ctypes.c_void_p()
        self._lib = L.lib()
        self.vocab, self.max_rows = vocab, max_rows
        L.check(self._lib.jev_logprobs_create(vocab, max_rows, device, ctypes.byref(self._h)))

    def close(self) -> None:
        if self._h:
            self._lib.jev_logprobs_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    @property
    def stream(self) -> int:
        """The handle's HIP stream (for graph capture or ordering by the caller)."""
        return int(self._lib.jev_logprobs_stream(self._h) or 0)

    def logprobs_device(self, logits: int, ld: int, rows: int, given: int = 0, n_given: int = 0, n_top: int = 0, temperature: float = 1.0,
                        logp: int = 0, entropy: int = 0, top: int = 0, top_logp: int = 0) -> None:
        """logits [rows][ld] -> logp [rows][n_given] of given, entropy [rows], top and top_logp [rows][n_top]; 0: not wanted."""
        L.check(self._lib.jev_logprobs_device(self._h, logits, ld, rows, given, n_given, n_top, temperature, logp, entropy, top, top_logp))

    def sync(self) -> None:
        """Waits for the handle's work."""
        L.check(self._lib.jev_logprobs_sync(self._h))
