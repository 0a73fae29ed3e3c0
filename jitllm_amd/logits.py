"""What is answered with beside the tokens: host mirror of jl_logprobs.

Behind the vocabulary projection of ``jitllm_amd.projections``, beside its ``argmaxLogits``::

    probabilities = LogProbabilities(ctx, maxRows, vocab, top=5)
    ...
    projections.projection(xb, logits, wcls, dim, vocab, False, rows)
    projections.argmaxLogits(logits, vocab, tokens, rows)
    probabilities.compute(logits, rows, tokens=tokens, logprobs=logprobs, topTokens=topTokens, topLogprobs=topLogprobs)

Every array lies on the device: a few numbers a row go to the host in place of its logits.
"""
from __future__ import annotations

from . import _lib as L
from .runtime import Context


def _array(name: str, array, count: int):
    if array.nbytes < 4 * count:
        raise ValueError(f"{name}: {count} values of 4 bytes in an array of {array.nbytes}")
    return array.ptr


class LogProbabilities:
    """Log probabilities over rows of ``vocab`` logits, with the workspace that a call's workgroups join in
    (jl_logprobs).  Calls that may run at the same time need one each.  ``top``: how many of the most probable
    tokens a call lists, at most 64.  ``maxRows`` is the caller's own note: the workspace is the same for any
    number of rows."""

    def __init__(self, ctx: Context, maxRows: int, vocab: int, top: int = 0):
        self.ctx, self._lib = ctx, ctx._lib
        self.maxRows, self.vocab, self.top = int(maxRows), int(vocab), int(top)
        nbytes = self._lib.jl_logprobs_workspace_bytes(self.vocab, self.top)
        if not nbytes or self.top > self.vocab:
            raise ValueError(f"the {top} most probable of {vocab} tokens (at most 64)")
        self.workspace = ctx.raw_buffer(nbytes)
        L.check(self._lib.jl_logprobs_workspace_init(ctx.handle, self.workspace.ptr, nbytes))

    def compute(self, logits, rows: int, tokens=None, logprobs=None, entropy=None, topTokens=None, topLogprobs=None,
                tokensPerRow: int = 1, scale: float = 1.0, cap: float = 0.0, rowStride: int | None = None) -> None:
        """``logprobs`` [rows x tokensPerRow] of ``tokens``, ``entropy`` [rows], ``topTokens`` and ``topLogprobs``
        [rows x top] of ``softmax(scale * x)``, x the logits or, where ``cap`` is positive, ``cap * tanh(logits /
        cap)``.  What is not given is not computed.  ``rowStride``: logits from a row to the next, ``vocab``
        unless given."""
        vocab = self.vocab
        stride = vocab if rowStride is None else rowStride
        if stride < vocab or (rows > 0 and logits.nbytes < 4 * ((rows - 1) * stride + vocab)):
            raise ValueError(f"{rows} rows of {vocab} logits, {stride} apart, in an array of {logits.nbytes} bytes")
        if (tokens is None) != (logprobs is None) or (topTokens is None) != (topLogprobs is None):
            raise ValueError("tokens without logprobs, or one of topTokens and topLogprobs without the other")
        per = tokensPerRow if tokens is not None else 0
        top = self.top if topTokens is not None else 0
        status = self._lib.jl_logprobs(
            self.ctx.handle, logits.ptr, rows, vocab, stride, scale, cap, _array("tokens", tokens, rows * per) if per else None, per,
            _array("logprobs", logprobs, rows * per) if per else None, _array("entropy", entropy, rows) if entropy is not None else None,
            top, _array("topTokens", topTokens, rows * top) if top else None,
            _array("topLogprobs", topLogprobs, rows * top) if top else None, self.workspace.ptr, self.workspace.nbytes)
        if status:
            L.check(status)
