"""How a beam search chooses. `BeamState` is what a batch of sequences keeps on the device between two choices; the choice
itself is `ops.beam_select` (csrc/beam_select.cu)."""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch


@dataclass(frozen=True)
class BeamOptions:
    beams: int = 4
    """Texts that are followed at a time, and results per prompt."""
    length_penalty: float = 1.0
    """A text's score is the sum of its tokens' log probabilities over (tokens) ** length_penalty, the stop token counted. A search
    takes penalties up to that at which its longest text would be divided by 2 ** 96 (about 8 for 2,000 tokens)."""
    early_stopping: bool = False
    """End as soon as `beams` texts have ended; otherwise only when no running text could do better than the worst of them at
    its present length."""

    MAX_BEAMS = 32

    def __post_init__(self) -> None:
        if not 1 <= self.beams <= self.MAX_BEAMS:
            raise ValueError(f"beams must be between 1 and {self.MAX_BEAMS}")
        if not 0 <= self.length_penalty < math.inf:  # (also refuses NaN)
            raise ValueError("length_penalty must be non-negative and finite")

    LARGEST_DIVISOR = 96
    """Scores are float32: divided by up to 2 ** 96 every sum of log probabilities that is not 0 stays a normal number."""

    def check_length(self, tokens: int) -> None:
        """Raises if texts of up to `tokens` tokens, and the stop token, have a score too small to be ordered by."""
        if self.length_penalty * math.log2(max(tokens, 0) + 1) > self.LARGEST_DIVISOR:
            raise ValueError(f"length_penalty {self.length_penalty} with texts of up to {tokens} tokens: scores would be divided by "
                             f"more than 2 ** {self.LARGEST_DIVISOR}")


class BeamState:
    """Device state of `sequences` searches: every beam's score, the texts that have ended (their scores, descending, and
    where each one ended: tokens before its stop token, and the beam), and whether a search is over."""

    def __init__(self, sequences: int, beams: int, device) -> None:
        self.scores = torch.zeros((sequences, beams), dtype=torch.float32, device=device)
        self.finished = torch.full((sequences, beams), -torch.inf, dtype=torch.float32, device=device)
        self.finished_at = torch.full((sequences, beams, 2), -1, dtype=torch.int32, device=device)
        self.done = torch.zeros(sequences, dtype=torch.int32, device=device)

    def tensors(self) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
        return self.scores, self.finished, self.finished_at, self.done

    def take(self, other: "BeamState", rows: list[int]) -> None:
        """This state becomes the given rows of `other`."""
        index = torch.tensor(rows, dtype=torch.long, device=self.scores.device)
        for mine, theirs in zip(self.tensors(), other.tensors()):
            mine.copy_(theirs[index])
