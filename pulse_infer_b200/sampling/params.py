"""Per-request sampling options, with the names and meanings the reference's generation demo uses
(``demo/qwen3_infer.cpp:229-239,590-592``), and beside them the logit rules that the reference does not have: repetition and
frequency penalty, biases, a grammar."""
from __future__ import annotations

import math
from dataclasses import dataclass

import numpy as np

F32_MAX, F32_TINY = (2.0 - 2.0 ** -23) * 2.0 ** 127, 2.0 ** -126       # largest and smallest normal number of 32 bits


@dataclass(frozen=True)
class SamplingParams:
    temperature: float = 0.0        # <= 0: greedy (qwen3_infer.cpp:277)
    top_k: int = 0                  # <= 0: all tokens (qwen3_infer.cpp:336)
    top_p: float = 0.0              # active only for 0 < p < 1 (qwen3_infer.cpp:395)
    presence_penalty: float = 0.0   # subtracted once from every token already in prompt or output (251-264)
    banned_tokens: tuple = ()       # never sampled (522-535)
    seed: int = 0                   # the draws of a request depend on (seed, index of the draw) only
    use_greedy: bool = False        # qwen3_infer.cpp:236
    # in the order in which they apply (ops.logit_rules): repetition, frequency, presence, biases and bans, grammar
    repetition_penalty: float = 1.0  # logits of tokens in prompt or output are divided by it if positive, else multiplied
    frequency_penalty: float = 0.0   # subtracted once for every time a token was generated
    logit_bias: tuple = ()           # (token, value) pairs, or {token: value}, that are added; -inf forbids the token
    # an object with ``token_mask(generated) -> None or ceil(vocabulary / 32) 32-bit words`` (bit v % 32 of word v / 32 set:
    # token v is allowed), asked before every token with the tokens generated so far
    grammar: object = None

    def __post_init__(self):
        # what the kernel cannot take is refused here: in a step it would stop the other requests too
        if not F32_TINY <= self.repetition_penalty <= F32_MAX:
            raise ValueError(f"repetition_penalty must be positive and finite in 32 bits, got {self.repetition_penalty}")
        if not abs(self.frequency_penalty) <= F32_MAX:
            raise ValueError(f"frequency_penalty must be finite in 32 bits, got {self.frequency_penalty}")
        try:
            pairs = self.logit_bias.items() if hasattr(self.logit_bias, "items") else self.logit_bias
            bias = tuple((int(t), float(v)) for t, v in pairs)
            banned = tuple(int(t) for t in self.banned_tokens)
        except (TypeError, ValueError, OverflowError) as exc:
            raise ValueError(f"logit_bias must hold (token, value) pairs and banned_tokens token ids: {exc}") from exc
        for token, value in bias:
            if not (abs(value) <= F32_MAX or value == -math.inf):
                raise ValueError(f"logit_bias of token {token} must be finite in 32 bits or -inf, got {value}")
        object.__setattr__(self, "logit_bias", bias)
        object.__setattr__(self, "banned_tokens", banned)
        if self.grammar is not None and not callable(getattr(self.grammar, "token_mask", None)):
            raise ValueError("a grammar needs a token_mask(generated) method")

    def token_mask(self, generated: list, vocab_size: int):
        """What the grammar allows behind ``generated``: ceil(vocab_size / 32) 32-bit words, or None for everything."""
        if self.grammar is None:
            return None
        mask = self.grammar.token_mask(generated)
        if mask is None:
            return None
        mask, words = np.array(mask).reshape(-1), (vocab_size + 31) // 32       # a copy: the grammar may fill its array again
        if mask.size != words or mask.dtype.itemsize != 4 or mask.dtype.kind not in "iu":
            raise ValueError(f"a token mask must hold {words} 32-bit words, got {mask.size} of {mask.dtype}")
        return mask.view(np.int32)

    @property
    def greedy(self) -> bool:
        return self.use_greedy or self.temperature <= 0.0

    @property
    def needs_history(self) -> bool:
        """Whether the tokens so far have a say in the next one."""
        return (self.presence_penalty > 0.0 or self.repetition_penalty != 1.0 or self.frequency_penalty != 0.0
                or self.grammar is not None)

    @property
    def needs_prompt_len(self) -> bool:
        """Whether it matters which of the tokens so far were generated."""
        return self.frequency_penalty != 0.0 or self.grammar is not None

    @property
    def edits_logits(self) -> bool:
        return self.needs_history or bool(self.banned_tokens) or bool(self.logit_bias)
