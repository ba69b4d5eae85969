"""What a model says of given tokens: their log probabilities, the entropy of the row they were drawn
from, and the most probable alternatives, on the device (``csrc/scores.cu``). The probabilities are
the model's own, of the whole vocabulary: no temperature and no filter is in them. The reference
returns chosen tokens only; scores are this library's own."""
from __future__ import annotations

import functools
from dataclasses import dataclass
from typing import List, Optional, Tuple

import torch

from .. import kernels as K
from ..errors import InferError


@functools.lru_cache(maxsize=64)
def _nothing(rows: int, device) -> Tuple[torch.Tensor, torch.Tensor]:
    """No alternatives' ids and log probabilities: tensors without a value."""
    return (torch.empty((rows, 0), dtype=torch.int32, device=device),
            torch.empty((rows, 0), dtype=torch.float32, device=device))


@dataclass
class TokenScore:
    """The scores of one token on the host: its log probability, the entropy of what it was chosen
    from, and the most probable ids with their log probabilities."""
    logprob: float
    entropy: float
    alternatives: List[Tuple[int, float]]


@dataclass
class Scores:
    """One entry a row: ``logprobs`` and ``entropy`` (natural logarithms, float32 [rows]); the ids
    (int32) and log probabilities of the alternatives [rows, top], the most probable first and the
    lowest id first among equals; negative infinities and NaNs come last, the lowest id first. A row
    with a NaN or a positive infinity among its logits, or with nothing but negative infinities, has
    no distribution: its numbers are NaN."""
    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_ids: torch.Tensor
    top_logprobs: torch.Tensor
    buffer: Optional[torch.Tensor] = None     # where all four lie one after another, if they do

    @classmethod
    def empty(cls, rows: int, top: int, device) -> "Scores":
        floats = torch.empty(rows * (2 + 2 * top), dtype=torch.float32, device=device)
        return cls.in_buffer(floats, rows, top)

    @classmethod
    def beside(cls, floats: torch.Tensor, ints: torch.Tensor, rows: int, top: int) -> "Scores":
        """Scores on the device of a float32 and an int32 tensor (four new tensors are made in less
        time than views of one)."""
        logprobs, entropy = floats.new_empty(rows), floats.new_empty(rows)
        if top == 0:
            return cls(logprobs, entropy, *_nothing(rows, floats.device))
        return cls(logprobs, entropy, ints.new_empty(rows, top), floats.new_empty(rows, top))

    @classmethod
    def in_buffer(cls, floats: torch.Tensor, rows: int, top: int) -> "Scores":
        """Scores that lie in a contiguous float32 tensor of ``rows * (2 + 2 * top)`` values one after
        another, so that one copy brings them elsewhere."""
        at, n = floats.storage_offset(), rows * top
        shape, step = (rows, top), (top or 1, 1)
        got = cls(floats.as_strided((rows,), (1,), at), floats.as_strided((rows,), (1,), at + rows),
                  floats.view(torch.int32).as_strided(shape, step, at + 2 * rows),
                  floats.as_strided(shape, step, at + 2 * rows + n))
        got.buffer = floats
        return got

    def rows(self, a: int, b: int) -> "Scores":
        """Rows a .. b - 1, in the same memory."""
        return Scores(self.logprobs[a:b], self.entropy[a:b], self.top_ids[a:b],
                      self.top_logprobs[a:b])

    def put(self, places: torch.Tensor, rows: "Scores") -> None:
        """``rows`` go to ``places`` (int64, on the device) of these."""
        for mine, theirs in zip(self.tensors(), rows.tensors()):
            mine.index_copy_(0, places, theirs)

    def take(self, rows: "Scores") -> None:
        """All of ``rows``, copied."""
        for mine, theirs in zip(self.tensors(), rows.tensors()):
            mine.copy_(theirs)

    def on_host(self) -> List["TokenScore"]:
        """One ``TokenScore`` a row (waits for the device)."""
        rows, top = self.top_ids.shape
        if self.buffer is not None:
            return Scores.in_buffer(self.buffer.cpu(), rows, top)._listed()
        return self._listed()

    def _listed(self) -> List["TokenScore"]:
        lp, en, ids, alt = (t.tolist() for t in self.tensors())
        return [TokenScore(a, b, list(zip(i, c))) for a, b, i, c in zip(lp, en, ids, alt)]

    def tensors(self):
        return self.logprobs, self.entropy, self.top_ids, self.top_logprobs


def candidates(vocab: int, vocab_limit: Optional[int]) -> int:
    """How many ids take part: all, or those below ``vocab_limit``."""
    if vocab_limit is None:
        return vocab
    if vocab_limit < 1:
        raise InferError(f"scores among the ids below {vocab_limit}")
    return min(vocab, vocab_limit)


def check_top(top: int, vocab: int) -> int:
    if type(top) is not int or not 0 <= top <= K.TOP_SCORES or top > vocab:
        raise InferError(f"{top} alternatives: 0 to {min(K.TOP_SCORES, vocab)} can be had")
    return top


def check_tokens(tokens: torch.Tensor, rows: int, device: int) -> None:
    if (tokens.dtype is not torch.int32 or tokens.dim() != 1 or tokens.numel() != rows
            or tokens.get_device() != device):
        raise InferError(f"scores of {rows} rows: tokens are {tokens.dtype} {tuple(tokens.shape)} on "
                         f"{tokens.device}, not int32 [{rows}] beside them")


def check_out(out: Scores, rows: int, top: int, device: int) -> None:
    for t, dtype, shape in zip(out.tensors(), (torch.float32, torch.float32, torch.int32, torch.float32),
                               ((rows,), (rows,), (rows, top), (rows, top))):
        if (t.dtype is not dtype or t.shape != shape or not t.is_contiguous()
                or t.get_device() != device):
            raise InferError(f"scores of {rows} rows and {top} alternatives into {t.dtype} "
                             f"{tuple(t.shape)} on {t.device}")


def check_score(h: torch.Tensor, tokens: torch.Tensor, top: int, hidden: int, vocab: int,
                vocab_limit: Optional[int]) -> int:
    """Refuses what a head of ``vocab`` rows of ``hidden`` values cannot score; how many ids take
    part."""
    if h.dim() != 2 or h.shape[1] != hidden or (hidden > 1 and h.stride(1) != 1):
        raise InferError(f"scores: the head's input is {tuple(h.shape)} with strides {h.stride()}, not "
                         f"rows of {hidden} values")
    vocab = candidates(vocab, vocab_limit)
    check_top(top, vocab)
    check_tokens(tokens, h.shape[0], h.get_device())
    return vocab


def token_scores(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0,
                 vocab_limit: Optional[int] = None, out: Optional[Scores] = None) -> Scores:
    """The scores of ``tokens`` (int32 [rows]) under ``logits`` (float32 [rows, vocab], both on the
    device; rows may lie apart). An id that is none of the vocabulary (-1 for "no token") scores NaN.
    ``top``: alternatives, up to 32. ``vocab_limit``: only the ids below it take part. ``out``: to
    write into, contiguous, as ``Scores.empty`` makes it. Runs on the current stream of the logits'
    device and reads nothing back; what it needs besides is allocated for the call alone."""
    shape = logits.shape
    if len(shape) != 2 or logits.dtype is not torch.float32 or shape[1] == 0:
        raise InferError(f"scores: logits are {logits.dtype} {tuple(shape)}, not float32 [rows, vocab]")
    rows, vocab = shape
    if vocab > 1 and logits.stride(1) != 1:
        raise InferError("scores: the logits of a row do not lie side by side")
    if vocab_limit is not None:
        vocab = candidates(vocab, vocab_limit)
    check_top(top, vocab)
    device = logits.get_device()
    check_tokens(tokens, rows, device)
    if out is None:
        out = Scores.beside(logits, tokens, rows, top)
    else:
        check_out(out, rows, top, device)
    if rows == 0:
        return out
    if not tokens.is_contiguous():
        tokens = tokens.contiguous()
    if K.elsewhere(device):
        with K.on_device_of(logits):
            K.token_scores(logits, vocab, tokens, top, out)
    else:
        K.token_scores(logits, vocab, tokens, top, out)
    return out
