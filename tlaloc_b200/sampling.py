"""How the next token of a request is drawn: the settings of `ops.sample` and the random numbers it takes.

The number of a draw is a function of the request's seed and of how many tokens it has produced, so a continuation depends neither on what else
runs beside it nor on a request that was sent back and read again.
"""
from __future__ import annotations

import hashlib
import struct
from dataclasses import dataclass

import numpy as np


@dataclass(frozen=True)
class Sampling:
    """temperature 0: the first maximum; top_k 0, top_p 1 and min_p 0 keep every token."""

    temperature: float = 1.0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0
    seed: int = 0

    def __post_init__(self):
        for name, fits, what in (("temperature", 0 <= self.temperature < float("inf"), "finite and not negative"), ("top_k", 0 <= self.top_k < 2**31, "in [0, 2^31)"),
                                 ("top_p", 0 <= self.top_p <= 1, "in [0, 1]"), ("min_p", 0 <= self.min_p <= 1, "in [0, 1]"),
                                 ("seed", -2**63 <= self.seed < 2**64, "an integer of 64 bits")):
            if not fits:
                raise ValueError(f"sampling: {name} is {what}, not {getattr(self, name)}")
        for name in ("top_k", "seed"):
            if int(getattr(self, name)) != getattr(self, name):
                raise ValueError(f"sampling: {name} is an integer, not {getattr(self, name)}")

    def uniform(self, index: int) -> float:
        """The random number of the request's draw `index`: 24 bits of a hash of (seed, index), a multiple of 2^-24 in [0, 1) that f32 holds exactly."""
        digest = hashlib.blake2b(struct.pack("<QQ", int(self.seed) % 2**64, index), digest_size=4).digest()
        return (int.from_bytes(digest, "little") >> 8) * 2.0**-24


GREEDY = Sampling(temperature=0.0)


def pack(draws) -> np.ndarray:
    """draws [(Sampling or None, index)] -> one int32 array [5, rows] to copy at once: uniforms, temperature, top_p and min_p (f32 bits), top_k."""
    out = np.zeros((5, len(draws)), np.int32)
    reals = out[:4].view(np.float32)
    for i, (s, index) in enumerate(draws):
        s = s or GREEDY
        reals[:, i] = (s.uniform(index), s.temperature, s.top_p, s.min_p)
        out[4, i] = s.top_k
    return out
