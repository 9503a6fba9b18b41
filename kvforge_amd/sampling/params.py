"""Per-request sampling parameters, names and meanings as in the reference
(src/tokenvault/sampling.py:18-37)."""

from __future__ import annotations

from dataclasses import dataclass, field


@dataclass
class SamplingParams:
    max_tokens: int = 64
    temperature: float = 1.0  # 0 = greedy
    top_k: int = 0  # 0 = disabled
    top_p: float = 1.0
    stop_token_ids: list[int] = field(default_factory=list)
    ignore_eos: bool = False
    # Stream of the counter-based generator; None = the request's arrival index.
    seed: int | None = None

    def __post_init__(self) -> None:
        if self.temperature < 0:
            raise ValueError("temperature must be >= 0")
        if not 0 < self.top_p <= 1:
            raise ValueError("top_p must be in (0, 1]")
        if self.max_tokens < 1:
            raise ValueError("max_tokens must be >= 1")
        if self.top_k < 0:
            raise ValueError("top_k must be >= 0")

    @property
    def greedy(self) -> bool:
        return self.temperature == 0.0


@dataclass
class BeamParams:
    """Parameters of a beam search.  ``width`` beams a request are followed, the best by the sum of their tokens' log-probabilities;
    one whose next token is a stop token ends, if it is among the ``width`` best of all continuations, and the ``width`` best of the
    others go on.  Ended beams are ranked by that sum over ``(number of output tokens) **
    length_penalty`` (the stop token counts).  A request is done once ``width`` beams have ended and, unless
    ``early_stopping``, no living beam's score so far beats the worst of them; or after ``max_tokens``, where the living ones
    end too.  ``num_return``: how many sequences are handed back, the best first (default: all ``width``)."""

    width: int = 4
    max_tokens: int = 64
    length_penalty: float = 1.0
    early_stopping: bool = False
    stop_token_ids: list[int] = field(default_factory=list)
    ignore_eos: bool = False
    num_return: int | None = None

    def __post_init__(self) -> None:
        if not 1 <= self.width <= 32:
            raise ValueError(f"a beam search follows 1 to 32 beams, got {self.width}")
        if self.max_tokens < 1:
            raise ValueError("max_tokens must be >= 1")
        if self.num_return is not None and not 1 <= self.num_return <= self.width:
            raise ValueError(f"num_return must be between 1 and the width ({self.width}), got {self.num_return}")
