"""What a model says about a token that stands at some place of a request: its log probability and its alternatives.

The numbers come from `ops.token_logprobs` and `ops.head_logprobs`, of the logits as the model gives them: before the repeat
penalty, the temperature and the other rules of a draw.
"""
from __future__ import annotations

from dataclasses import dataclass, field

import numpy as np
import torch

MAX_ALTERNATIVES = 64


@dataclass
class TokenScore:
    token: int
    logprob: float
    entropy: float                     # of the distribution the token is one outcome of, in nats
    rank: int | None = None            # how many tokens were more likely (None where it was not asked for)
    top: list = field(default_factory=list)      # the most likely tokens, [(id, log probability)]


def check_alternatives(n: int, vocab: int) -> int:
    n = int(n)
    if not 0 <= n <= min(MAX_ALTERNATIVES, vocab):
        raise ValueError(f"{n} alternatives per token are not 0..{min(MAX_ALTERNATIVES, vocab)}")
    return n


class ScoreRows:
    """The results of `rows` tokens in one block of 32-bit words, so that they travel to the host in one copy:
    log probabilities | entropies | ranks | ids [rows, top] | log probabilities of those [rows, top]."""

    def __init__(self, flat: torch.Tensor, rows: int, top: int):
        self.flat, self.rows, self.top = flat[:self.words(rows, top)], rows, top
        part = [flat[i * rows:(i + 1) * rows] for i in range(3)]
        self.logprob, self.entropy, self.rank = part[0].view(torch.float32), part[1].view(torch.float32), part[2]
        n = rows * top
        self.ids = flat[3 * rows:3 * rows + n].view(rows, top) if top else None
        self.top_logprobs = flat[3 * rows + n:3 * rows + 2 * n].view(torch.float32).view(rows, top) if top else None

    @staticmethod
    def words(rows: int, top: int) -> int:
        return rows * (3 + 2 * top)

    @staticmethod
    def parse(words: np.ndarray, rows: int, top: int, tokens, keep=None) -> list[TokenScore]:
        """The rows of a block that has reached the host; `tokens[i]` is the token of row i, `keep[i]` how many alternatives it wants."""
        f = words.view(np.float32)
        n = rows * top
        ids = words[3 * rows:3 * rows + n].reshape(rows, top)
        lps = f[3 * rows + n:3 * rows + 2 * n].reshape(rows, top)
        out = []
        for i, tok in enumerate(tokens):
            k = top if keep is None else keep[i]
            rank = int(words[2 * rows + i])
            out.append(TokenScore(int(tok), float(f[i]), float(f[rows + i]), rank if rank >= 0 else None,
                                  [(int(a), float(b)) for a, b in zip(ids[i, :k], lps[i, :k])]))
        return out
