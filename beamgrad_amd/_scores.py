# SPDX-License-Identifier: MIT
"""Log-probabilities of given tokens under rows of logits, on the GPU: the
teacher-forced scores that :func:`sequence_scores` and the ``rescore_fn`` of
:func:`beam_search` take, with the entropy of each row, its most likely tokens, and
a gradient.

A row of logits is read once, and nothing of its size is stored but, in a backward
pass, its gradient: no log-softmax of the rows exists. The C entries are in
``include/beamgrad_score.h``. The reference has no counterpart: its re-scoring
gathers from log-probabilities that its caller computes (reference
python/beamgrad/_search.py:314-327).
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from ._torch import _ops as _torch_ops

_forward = _torch_ops.token_logprobs.default
_backward = _torch_ops.token_logprobs_backward.default


class TokenLogprobs(NamedTuple):
    """What :func:`token_logprobs` returns; ``None`` for what was not asked for."""

    logprobs: torch.Tensor  # [...] float32: of the given tokens
    entropy: torch.Tensor | None  # [...] float32: of each row
    top_logprobs: torch.Tensor | None  # [..., top] float32, largest first
    top_tokens: torch.Tensor | None  # [..., top] int64


def _register() -> None:
    """Shape-only forms, and vmap rules: the leading dimensions are whatever they
    are, so a vmapped one is one more of them."""

    def forward(logits, tokens, top, entropy, stats):
        shape, f32 = tuple(tokens.shape), torch.float32
        return (logits.new_empty(shape, dtype=f32), logits.new_empty(shape if entropy else (*shape, 0), dtype=f32),
                logits.new_empty((*shape, top), dtype=f32), logits.new_empty((*shape, top), dtype=torch.int64),
                logits.new_empty((*shape, 4 if stats else 0), dtype=f32))

    def backward(logits, *_args):
        return logits.new_empty(logits.shape)

    def lead(t, dim, n):
        if t is None:
            return None
        return t.unsqueeze(0).expand(n, *t.shape) if dim is None else t.movedim(dim, 0)

    def forward_rule(info, in_dims, logits, tokens, top, entropy, stats):
        n = info.batch_size
        return _forward(lead(logits, in_dims[0], n), lead(tokens, in_dims[1], n), top, entropy, stats), (0,) * 5

    def backward_rule(info, in_dims, *args):
        return _backward(*(lead(t, d, info.batch_size) for t, d in zip(args, in_dims, strict=True))), 0

    torch.library.register_fake("beamgrad::token_logprobs", forward)
    torch.library.register_fake("beamgrad::token_logprobs_backward", backward)
    torch.library.register_vmap("beamgrad::token_logprobs", forward_rule)
    torch.library.register_vmap("beamgrad::token_logprobs_backward", backward_rule)


_register()


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, top: int = 0, entropy: bool = False) -> TokenLogprobs:
    """``log_softmax(logits)`` at the given tokens.

    ``logits`` is ``[..., V]`` (float32, float16 or bfloat16), ``tokens`` ``[...]``
    (int32 or int64). A row whose token lies outside ``[0, V)`` (a search's sequences
    end in -1) is not read: its log-probability and entropy are 0, it has no
    alternatives (-1, at -inf) and its gradient is zeros, so sums over a sequence
    need no mask. With ``top`` (up to 64) the ``top`` most likely tokens of each row
    and their log-probabilities are returned, of equally likely ones the lowest
    first; with ``entropy`` ``-sum(p log p)``.

    Sums are held in 32 bits, whatever the logits' type. Where all of a row is -inf
    its log-probabilities are -inf, its entropy is 0 and its gradient zeros; a row that
    holds NaN or +inf is NaN throughout (its alternatives -1). The results are
    differentiable (the log-probabilities, the alternatives' and the entropy), once,
    in reverse mode; the gradient has the logits' type, rounded once.

    As a rescoring of a search's final beams::

        def rescore(sequences, lengths):
            return token_logprobs(model(sequences), sequences).logprobs
    """
    for name, t in (("logits", logits), ("tokens", tokens)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if isinstance(top, bool) or not isinstance(top, int):
        raise TypeError(f"top must be an int, got {type(top).__name__}")
    lp, h, best, which, _stats = _forward(logits, tokens, top, bool(entropy), False)
    return TokenLogprobs(lp, h if entropy else None, best if top else None, which if top else None)
