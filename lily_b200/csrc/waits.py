"""The waits that kernels of this process gave up, as the host has heard of them.

A kernel whose bounded wait runs out says so in a word of the host's memory, makes its outputs NaN and ends.  The kernels of a kind share one word,
which its reader clears, and it does not say whose step it was: so everybody who uses them hears of each, whoever read the word.
"""

from __future__ import annotations

import threading


class Lost:
    """The waits of one kind of kernel."""

    def __init__(self):
        self.lock = threading.Lock()
        self.count = self.row = 0

    def heard(self, read) -> int:
        """How many there were, after a look at the word by ``read``; ``row`` is what it held last."""
        with self.lock:
            found = read()
            if found:
                self.count += 1
                self.row = found
            return self.count


DECODE = Lost()                  # decode attention (ops.attention_decode_lost)
KEY_WEIGHTS = Lost()             # column sums of prompt portions (ops.key_weights_lost)
LINEAR4 = Lost()                 # products with 4-bit weights on tcgen05 (ops.linear4_lost)


class Listener:
    """What one user of attention that weighs its keys has heard; nothing of what was lost before it was made."""

    def __init__(self, ops):
        self.ops, self.decode, self.key_weights = ops, DECODE.count, KEY_WEIGHTS.count

    def check(self) -> None:
        """Raises, once for each, when a kernel that the host has waited for gave up a wait.  (Two words in the host's memory are read.)"""
        decode = getattr(self.ops, "attention_decode_lost", None)               # (stand-ins for the kernels wait for nothing)
        weights = getattr(self.ops, "key_weights_lost", None)
        heard = (DECODE.heard(decode) if decode else self.decode, KEY_WEIGHTS.heard(weights) if weights else self.key_weights)
        was, (self.decode, self.key_weights) = (self.decode, self.key_weights), heard
        if heard[0] != was[0]:
            raise RuntimeError(f"decode attention: a tile of keys did not arrive in time (row {DECODE.row - 1} of its step); the step's outputs and weights are void")
        if heard[1] != was[1]:
            raise RuntimeError(f"column sums of a portion: a wait was given up (code {KEY_WEIGHTS.row >> 24}, block {KEY_WEIGHTS.row & 0xFFFFFF}); the portion's weights are void")


__all__ = ["DECODE", "KEY_WEIGHTS", "LINEAR4", "Listener", "Lost"]
