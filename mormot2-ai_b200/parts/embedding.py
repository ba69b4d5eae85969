"""Token embedding (rows of the table into the float32 residual, times ``scale`` where a
design names one; the reference scales nothing: ``decoder.pas:3292-3309``) and the head (logits = h · Headᵀ in float32, the
head being the embedding when tied: ``model.qwen3.pas:555-579``; a head with ``scale``
multiplies its float32 logits by that constant; one with ``softcap`` c turns them into
c tanh(logits / c))."""
from __future__ import annotations

from typing import Dict, List, Optional

import torch

from .. import kernels as K
from ..errors import InferError
from ..sampling.scores import Scores, check_score
from .base import EMBEDDINGS, ENTRIES, HEADS, Part, TensorNeed
from .linear import Linear, Pending


# Logits of rows whose scores go through memory: so many values at a time (1 GiB)
SCORE_BAND = 1 << 28


def scores_through_memory(rows: int, vocab: int, top: int) -> bool:
    """Whether the logits of these rows are better stored: those of few rows with many alternatives. The
    fused kernel keeps lists of its own for every strip of a row, while the stored logits of few rows are
    read from L2. Fused | stored, us: 20 alternatives of 151,936 ids, 32 rows of 1,024 values 93 | 88, 96
    rows 94 | 113; of 32,000 ids, 257 rows 72 | 57, 512 rows 80 | 70, 1,001 rows 97 | 117; 32
    alternatives of 151,936, 128 rows 129 | 117, 257 rows 201 | 201, of 2,560 values 291 | 330. (No bound on the
    values alone has both the 96 rows and the 512 on their quicker side; the 512 are not.) With 8 or
    fewer the fused kernel is as quick from the first row on: 5 alternatives, 8 rows of 1,024 values
    78 | 84, of 4,096 214 | 223, 128 rows of 1,024 84 | 109."""
    return rows * vocab <= (top - 8) << 20


class TokenEmbedding(Part):
    capturable = True

    def __init__(self, spec, prefix: str = ""):
        super().__init__(spec, prefix)
        self.name = spec.params["name"]
        self.vocab, self.hidden = int(spec.params["vocab_size"]), int(spec.params["hidden_size"])
        self.scale = float(spec.params.get("scale", 1.0))

    def tensors(self) -> List[TensorNeed]:
        return [TensorNeed(self.name, (self.vocab, self.hidden), "table")]

    def bind(self, weights: Dict[str, torch.Tensor], rt) -> None:
        self.table = weights[self.name]

    def forward(self, ids: torch.Tensor, x: torch.Tensor) -> None:
        """x [T, hidden], or [streams, T, hidden]: every stream starts as the same rows."""
        K.embed(self.table, ids, x, self.scale)


class LmHead(Part):
    capturable = True

    def __init__(self, spec, prefix: str = ""):
        super().__init__(spec, prefix)
        p = spec.params
        self.tied = bool(p["tied"])
        self.name = p["tied_to"] if self.tied else p["name"]
        self.stored_name = p["name"]
        self.vocab, self.hidden = int(p["vocab_size"]), int(p["hidden_size"])
        self.scale = float(p.get("scale", 1.0))
        self.softcap = float(p.get("softcap") or 0.0)    # logits <- c tanh(logits / c)

    def tensors(self) -> List[TensorNeed]:
        if self.tied:
            # a stored copy of a tied head is tolerated when it equals the embedding
            return [TensorNeed(self.stored_name, (self.vocab, self.hidden), "table", optional=True,
                               must_equal=self.name)]
        return [TensorNeed(self.name, (self.vocab, self.hidden), "matrix")]

    def bind(self, weights: Dict[str, torch.Tensor], rt) -> None:
        self.linear = Linear(weights[self.name], rt)

    def forward(self, h: torch.Tensor) -> torch.Tensor:
        logits = self.linear(h, out_dtype=torch.float32)
        if self.scale != 1.0:
            K.scale_rows(logits, self.scale)
        if self.softcap > 0:
            K.softcap_rows(logits, self.softcap)
        return logits

    def libraries(self, rt):
        return ["scores", "head_scores"] if rt.fast_kernels else ["scores"]

    def score(self, h: torch.Tensor, tokens: torch.Tensor, top: int = 0,
              vocab_limit: Optional[int] = None) -> Scores:
        """The scores of ``tokens`` (int32 [rows]) under the logits of ``h`` [rows, hidden], as
        ``token_scores`` of ``forward(h)`` gives them. Of more than a few bfloat16 rows the logits are
        never stored (``csrc/head_scores.cu``); others go through memory, a band of rows at a time."""
        limit = check_score(h, tokens, top, self.hidden, self.vocab, vocab_limit)
        if K.elsewhere(h.get_device()):
            with K.on_device_of(h):
                return self.score(h, tokens, top, vocab_limit)
        rows, weight, rt = h.shape[0], self.linear.weight, self.linear.rt
        if weight.get_device() != h.get_device():
            raise InferError(f"scores: the head's input is on {h.device}, its weight on {weight.device}")
        if not self.hidden <= h.stride(0) < 1 << 31:      # one row many times, or rows 4 GiB apart
            h = h.clone(memory_format=torch.contiguous_format)
        floats = h if h.dtype == torch.float32 else rt.workspace
        if floats is None:
            out = Scores.empty(rows, top, h.device)
        else:
            out = Scores.beside(floats, tokens, rows, top)
        if rows == 0:
            return out
        tokens = tokens.contiguous()
        if (self.linear.fast is not None and not scores_through_memory(rows, limit, top)
                and K.head_scores_supported(h, weight)):
            K.head_scores(h, weight, limit, self.scale, self.softcap, tokens, top, out, rt.error_word)
            return out
        band = max(256, SCORE_BAND // self.vocab)
        if rows <= band:
            K.token_scores(self.forward(h), limit, tokens, top, out)
            return out
        for a in range(0, rows, band):
            b = min(rows, a + band)
            K.token_scores(self.forward(h[a:b]), limit, tokens[a:b], top, out.rows(a, b))
        return out


class PassInput(Part):
    """What a pass through looped layers adds to the residual before its first layer: row
    ``row`` of the table ``name`` [rows, size] and, with ``add_embedding``, the embedding's
    output once more (the model keeps a copy of it for the runs that ask)."""
    capturable = True

    def __init__(self, spec, prefix: str = ""):
        super().__init__(spec, prefix)
        p = spec.params
        self.name = prefix + p["name"]
        self.rows, self.row, self.size = int(p["rows"]), int(p["row"]), int(p["size"])
        self.add_embedding = bool(p.get("add_embedding", False))

    def tensors(self) -> List[TensorNeed]:
        return [TensorNeed(self.name, (self.rows, self.size), "bias")]

    def bind(self, weights: Dict[str, torch.Tensor], rt) -> None:
        self.vector = weights[self.name][self.row].contiguous()

    def forward(self, x: torch.Tensor, x0) -> None:
        K.pass_input(x, self.vector, x0 if self.add_embedding else None)


class PassProjection(Part):
    """What a pass through looped layers starts from: x = W_in [x ; x0] + step[row], x0 the
    embedding's output (``names``: ``in`` [size, 2 size], x's columns first, and ``step`` [rows,
    size]). One kernel adds what is still pending into x, writes [x ; x0] in the activation type
    (x0 from the embedding's table) and puts step[row] in x's place; the product is added onto
    that."""
    capturable = True
    accepts_pending = True      # forward(..., pending=) -> what is pending afterwards

    def __init__(self, spec, prefix: str = ""):
        super().__init__(spec, prefix)
        p = spec.params
        self.names = {k: prefix + v for k, v in p["names"].items()}
        self.rows, self.row, self.size = int(p["rows"]), int(p["row"]), int(p["size"])

    def tensors(self) -> List[TensorNeed]:
        return [TensorNeed(self.names["in"], (self.size, 2 * self.size)),
                TensorNeed(self.names["step"], (self.rows, self.size), "bias")]

    def bind(self, weights: Dict[str, torch.Tensor], rt) -> None:
        self.rt = rt
        self.linear = Linear(weights[self.names["in"]], rt)
        self.vector = weights[self.names["step"]][self.row].to(torch.float32).contiguous()

    def forward(self, x: torch.Tensor, step, embedding, pending=None):
        from .block import BranchSums, settle
        if pending is not None and not isinstance(pending, BranchSums):
            settle(x, pending)
            pending = None
        both = torch.empty((x.shape[0], 2 * self.size), dtype=self.rt.dtype, device=x.device)
        K.pass_concat(x, pending.terms if pending is not None else [], embedding.table,
                      step.tok_ids, embedding.scale, self.vector, both)
        y = self.linear(both, out_dtype=torch.float32, defer="any")
        return BranchSums([(y.partial if isinstance(y, Pending) else y, 1.0, None)])


EMBEDDINGS.register("token_embedding", TokenEmbedding)
ENTRIES.register("pass_input", PassInput)
ENTRIES.register("pass_projection", PassProjection)
HEADS.register("lm_head", LmHead)
