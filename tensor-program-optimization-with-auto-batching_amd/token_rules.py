"""Rules for the tokens of a request - penalties for repeated tokens, biases, a grammar -, and their device arrays for a batch."""
from __future__ import annotations

import dataclasses
from typing import Callable, Iterable, Mapping, Optional, Sequence

import numpy as np
import torch

from . import ops


@dataclasses.dataclass(frozen=True)
class TokenRules:
    """What a request's answer is held to, applied to its logits ahead of the greedy choice (formulas: ops.constrained_argmax).
    repetition divides (multiplies, below zero) the logits of tokens that the prompt or the answer holds, presence and frequency are
    subtracted once and per occurrence from those that the answer holds, bias adds to tokens by id.  grammar(answer so far) names the
    token ids that may come next (None: all); where it leaves none, the answer ends."""
    repetition: float = 1.0
    presence: float = 0.0
    frequency: float = 0.0
    bias: Optional[Mapping[int, float]] = None
    grammar: Optional[Callable[[Sequence[int]], Optional[Iterable[int]]]] = None

    def __post_init__(self):
        if not self.repetition > 0:
            raise ValueError(f"TokenRules: repetition {self.repetition} is not positive")


class BatchRules:
    """The rules of a batch's rows (None: a row without), whose chosen tokens go on behind their histories."""

    def __init__(self, rules, prompts, answers, room, vocab, device):
        """prompts, answers: token ids per row; room: tokens a row may still be given (its history has no place for more); vocab: columns
        of the logits."""
        self.rules, self.vocab, self.device, self.left = [r or TokenRules() for r in rules], vocab, device, max(room, 1)
        for r in self.rules:
            if r.bias and not all(0 <= int(v) < vocab for v in r.bias):
                raise ValueError(f"TokenRules: a bias for a token outside 0..{vocab - 1}")
        B = len(self.rules)
        lens = [len(p) + len(a) for p, a in zip(prompts, answers)]
        history = np.full((B, max(lens, default=0) + max(room, 1)), -1, dtype=np.int32)
        for row, p, a in zip(history, prompts, answers):
            row[:len(p)], row[len(p):len(p) + len(a)] = p, a
        i32 = lambda a: torch.as_tensor(np.asarray(a, dtype=np.int32)).to(device)
        f32 = lambda n: torch.tensor([float(getattr(r, n)) for r in self.rules], dtype=torch.float32, device=device)
        args = dict(history=i32(history), lengths=i32(lens), gen_start=i32([len(p) for p in prompts]), append=True,
                    repetition=f32("repetition"), presence=f32("presence"), frequency=f32("frequency"))
        n = max((len(r.bias or ()) for r in self.rules), default=0)
        if n:
            ids, values = np.full((B, n), -1, np.int32), np.zeros((B, n), np.float32)
            for b, r in enumerate(self.rules):
                for j, (v, x) in enumerate((r.bias or {}).items()):
                    ids[b, j], values[b, j] = v, x
            args.update(bias_ids=i32(ids), bias=torch.from_numpy(values).to(device))
        self.held = [b for b, r in enumerate(self.rules) if r.grammar is not None]
        if self.held:
            self._words = np.zeros((len(self.held), -(-vocab // 32)), dtype=np.uint32)
            self.masks, self.mask_row = i32(self._words.view(np.int32)), i32(np.full(B, -1))
            args.update(masks=self.masks, mask_row=self.mask_row)
            self.allow(answers)
        self.args = ops.LogitRules(**args)

    def allow(self, answers):
        """Asks the grammars which tokens may come behind the rows' answers (ahead of the step that chooses them)."""
        rows = np.full(len(self.rules), -1, dtype=np.int32)
        for m, b in enumerate(self.held):
            allowed = self.rules[b].grammar(list(answers[b]))
            if allowed is None:
                continue
            v = np.unique(np.fromiter((int(x) for x in allowed), dtype=np.int64))
            if v.size and (v[0] < 0 or v[-1] >= self.vocab):
                raise ValueError(f"TokenRules: a grammar allows token {v[0] if v[0] < 0 else v[-1]} of {self.vocab}")
            self._words[m] = 0
            np.bitwise_or.at(self._words[m], v // 32, np.uint32(1) << (v % 32).astype(np.uint32))
            rows[b] = m
        if self.held:
            self.masks.copy_(torch.from_numpy(self._words.view(np.int32)))
            self.mask_row.copy_(torch.from_numpy(rows))

    def take(self):
        """Ahead of a step, recorded or not, that chooses tokens: a place of the histories is used."""
        if self.left <= 0:
            raise RuntimeError("BatchRules: no room for another token")
        self.left -= 1

    def choose(self, logits, out=None):
        """The rows' tokens [B] int32, -1 where none is left; they go behind the rows' histories."""
        return ops.constrained_argmax(logits, self.args, ids=out)
